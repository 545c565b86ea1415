// Host-only check of which decode units read their adopted prompts shared (no GPU needed): the form that was
// measured the faster one.  Linked against libsslm_hip.so; prints "ok" on success.
#include <algorithm>
#include <cstdio>

#include "../superslm_amd/csrc/batch_ops.h"

using namespace sslm_launch;

static int bad = 0;
struct Shape {
	int heads, kv, dim;
};
// `adopters` of a prompt of `prompt` positions with 32 of their own beside `loose` rows of `width` without one, 256 CUs
static void expect(bool want, Shape s, int adopters, int64_t prompt, int loose = 0, int64_t width = 0, bool per_head = false) {
	SharedUnit u{adopters + loose, s.heads, s.kv, s.dim, std::max(prompt + 33, width), adopters * prompt, adopters * 33 + loose * width, per_head};
	if (shared_attn_pays(u, 256) != want) {
		printf("FAIL %d/%dx%d, %d of %ld + %d of %ld: %d\n", s.heads, s.kv, s.dim, adopters, (long)prompt, loose, (long)width, !want);
		++bad;
	}
}

int main() {
	const Shape q7{28, 4, 128}, q1{12, 2, 128}, h8{32, 8, 128}, h8n{32, 8, 64}, h16{32, 16, 128}, g2{16, 8, 128}, wide{16, 4, 256};
	// adopters alone: by their length, one row, or few dims, later
	for (const Shape& s : {q7, q1})
		for (int n : {2, 4, 8, 16, 32}) {
			expect(false, s, n, 1000);
			expect(true, s, n, 2700);
			expect(true, s, n, 8000);
		}
	expect(false, q7, 1, 2600);
	expect(false, q7, 1, 3000);
	expect(true, q7, 1, 3400);
	expect(false, h8n, 1, 3300);
	expect(false, h8n, 2, 2700);
	expect(true, h8n, 2, 4000);
	expect(true, h8n, 8, 4000);
	expect(true, wide, 2, 2700);
	// a short prompt beside long rows without one: by what those take on every CU
	expect(true, q7, 1, 20, 3, 3000);
	expect(true, q7, 1, 20, 7, 3000);
	expect(false, q7, 1, 20, 15, 3000);
	expect(false, q7, 1, 20, 31, 3000);
	expect(false, q7, 1, 20, 23, 4000);
	expect(false, q7, 1, 20, 31, 4400);
	expect(false, q7, 8, 4000, 24, 4000);
	expect(false, q7, 1, 20, 63, 1000);
	expect(true, q1, 1, 20, 15, 3000);
	expect(true, q1, 1, 20, 15, 8000);
	expect(true, q1, 1, 20, 31, 4000);
	expect(false, q1, 1, 20, 47, 3000);
	expect(false, q1, 1, 20, 63, 4000);
	expect(false, q1, 1, 20, 127, 1000);
	expect(false, q1, 16, 4000, 48, 4000);
	// where one block per query head would run instead
	expect(true, q7, 1, 20, 39, 3600, true);
	expect(true, q7, 1, 20, 63, 4400, true);
	expect(true, q1, 1, 20, 127, 6000, true);
	// past one block per CU
	expect(true, q7, 1, 20, 95, 200, true);
	expect(true, q7, 24, 1000, 72, 1000, true);
	expect(true, q7, 1, 20, 127, 1000, true);
	expect(true, q7, 65, 32, 0, 0, true);
	expect(true, h8, 100, 32, 0, 0, true);
	expect(false, h8, 33, 300);
	expect(false, h8, 64, 300);
	expect(true, h8, 64, 1000);
	expect(false, h8, 1, 20, 32, 50);
	expect(false, h8, 1, 20, 63, 1000);
	expect(false, h8n, 65, 32, 0, 0, true);
	expect(true, h8n, 128, 32, 0, 0, true);
	expect(false, h8n, 1, 20, 64, 300, true);
	expect(true, h16, 33, 1000);
	expect(true, h16, 64, 1000);
	expect(false, h16, 1, 20, 99, 1000, true);
	expect(false, g2, 100, 32, 0, 0, true);
	expect(true, g2, 100, 1200, 0, 0, true);
	expect(false, g2, 1, 20, 99, 1000, true);
	expect(false, wide, 65, 32, 0, 0, true);
	expect(false, wide, 1, 20, 127, 300, true);
	if (bad) return 1;
	printf("ok\n");
	return 0;
}
