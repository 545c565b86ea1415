// Host-only check of which decode units read their adopted prompts shared (no GPU needed): the form that was
// measured the faster one.  Linked against libsslm_hip.so; prints "ok" on success.
#include <cstdio>

#include "../superslm_amd/csrc/batch_ops.h"

using sslm_launch::shared_attn_pays;

static int bad = 0;
// `adopters` of a prompt of `prompt` positions with 32 of their own beside `loose` rows of `width` without one, 256 CUs
static void expect(bool want, int kv, int adopters, int64_t prompt, int loose, int64_t width, bool per_head = false) {
	const int64_t own = adopters * 33 + loose * width, longest = prompt + 33 > width || !loose ? prompt + 33 : width;
	if (shared_attn_pays(adopters + loose, kv, longest, own, per_head, 256) != want) {
		printf("FAIL %d KV heads, %d of %ld + %d of %ld: %d\n", kv, adopters, (long)prompt, loose, (long)width, !want);
		++bad;
	}
}

int main() {
	// adopters alone: by their length, one row later than several
	for (int kv : {2, 4})
		for (int n : {2, 4, 8, 16, 32}) {
			expect(false, kv, n, 1000, 0, 0);
			expect(true, kv, n, 2700, 0, 0);
			expect(true, kv, n, 8000, 0, 0);
		}
	expect(false, 4, 1, 2600, 0, 0);
	expect(false, 4, 1, 3000, 0, 0);
	expect(true, 4, 1, 3400, 0, 0);
	// a short prompt beside long rows without one: by what those take on every CU
	expect(true, 4, 1, 20, 3, 3000);
	expect(true, 4, 1, 20, 7, 3000);
	expect(false, 4, 1, 20, 15, 3000);
	expect(false, 4, 1, 20, 31, 3000);
	expect(false, 4, 1, 20, 23, 4000);
	expect(false, 4, 1, 20, 31, 4400);
	expect(false, 4, 8, 4000, 24, 4000);
	expect(false, 4, 1, 20, 63, 1000);
	expect(true, 2, 1, 20, 15, 3000);
	expect(true, 2, 1, 20, 15, 8000);
	expect(true, 2, 1, 20, 31, 4000);
	expect(false, 2, 1, 20, 47, 3000);
	expect(false, 2, 1, 20, 63, 4000);
	expect(false, 2, 1, 20, 127, 1000);
	expect(false, 2, 16, 4000, 48, 4000);
	// where one block per query head would run instead, and past one block per CU
	expect(true, 4, 1, 20, 39, 3600, true);
	expect(true, 4, 1, 20, 63, 4400, true);
	expect(true, 2, 1, 20, 127, 6000, true);
	expect(true, 4, 1, 20, 95, 200);
	expect(true, 4, 24, 1000, 72, 1000);
	expect(true, 4, 1, 20, 127, 1000);
	if (bad) return 1;
	printf("ok\n");
	return 0;
}
