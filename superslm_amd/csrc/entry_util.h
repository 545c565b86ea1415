// What the C entries of the operators over device buffers share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/sslm_hip.h"
#include "kernels.h"

namespace sslm_launch {

constexpr int kMaxRows = 65535;  // a grid's y extent

inline size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// A launch on the caller's stream: the stream belongs to the current device, and nothing throws
// past the boundary.
template <typename F>
sslm_status on_stream(void* stream, F&& launch) {
	int cur = -1;
	hipDevice_t of = -1;
	if (hipGetDevice(&cur) != hipSuccess) return SSLM_INVALID_ARGUMENT;
	if (stream && (hipStreamGetDevice((hipStream_t)stream, &of) != hipSuccess || of != cur)) return SSLM_INVALID_ARGUMENT;
	(void)hipGetLastError();  // an error left by an unrelated earlier call is not this call's
	try {
		launch((hipStream_t)stream);
	} catch (const LaunchRefused& e) {
		fprintf(stderr, "sslm_hip: launch refused (%s)\n", e.what);
		return SSLM_HIP_LAUNCH_FAILED;
	} catch (...) {
		return SSLM_HIP_LAUNCH_FAILED;
	}
	return hipGetLastError() == hipSuccess ? SSLM_OK : SSLM_HIP_LAUNCH_FAILED;
}

inline bool workspace_ok(const void* ws, size_t have, size_t need, sslm_status* st) {
	*st = !ws ? SSLM_INVALID_ARGUMENT : (((uintptr_t)ws % 256) ? SSLM_MISALIGNED_BUFFER : SSLM_BUFFER_TOO_SMALL);
	return ws && (uintptr_t)ws % 256 == 0 && have >= need;
}

}  // namespace sslm_launch
