// batch_ops_graph_check.cpp's check over batches whose attention runs in the launches by planes, which hand each other
// their maxima, sums and contexts through the call's workspace: rows of more positions, and heads of more dims, than the
// one-launch form takes.  Prints "ok" on success.
#define main batch_ops_graph_check_main
#include "batch_ops_graph_check.cpp"
#undef main

int main() {
	Batch b[2];
	// 13 x 6 query rows to a prompt and KV head, two blocks; and heads of 256 dims
	b[0].rows = 40, b[0].heads = 12, b[0].kv = 2, b[0].dim = 128, b[0].prefixes = 3, b[0].n = 256, b[0].vocab = 500, b[0].adapters = 2;
	b[0].longest = 1500, b[0].own = 90;
	b[1].rows = 23, b[1].heads = 8, b[1].kv = 2, b[1].dim = 256, b[1].prefixes = 1, b[1].n = 64, b[1].vocab = 500, b[1].adapters = 2;
	b[1].longest = 300, b[1].own = 20;
	hipStream_t s[2];
	hipEvent_t fork, join;
	CK(hipEventCreateWithFlags(&fork, hipEventDisableTiming));
	CK(hipEventCreateWithFlags(&join, hipEventDisableTiming));
	for (int i = 0; i < 2; ++i) {
		b[i].make();
		CK(hipStreamCreateWithFlags(&s[i], hipStreamNonBlocking));
	}
	hipGraphExec_t one[2], both;
	for (int i = 0; i < 2; ++i) one[i] = capture(s[i], [&] { b[i].enqueue(b[i].out, s[i]); });
	both = capture(s[0], [&] {
		CK(hipEventRecord(fork, s[0]));
		CK(hipStreamWaitEvent(s[1], fork, 0));
		for (int i = 0; i < 2; ++i) b[i].enqueue(b[i].out, s[i]);
		CK(hipEventRecord(join, s[1]));
		CK(hipStreamWaitEvent(s[0], join, 0));
	});
	int live = 0;
	for (int round = 0; round < 4; ++round) {
		for (auto& x : b) {
			x.fill();
			x.ref.spoil();
			x.enqueue(x.ref, nullptr);
			CK(hipDeviceSynchronize());
			x.ref.down();
		}
		for (int how = 0; how < 3; ++how) {
			for (auto& x : b) x.out.spoil();
			if (how == 0)
				for (int i = 0; i < 2; ++i) b[i].enqueue(b[i].out, s[i]);
			else if (how == 1)
				for (int i = 0; i < 2; ++i) CK(hipGraphLaunch(one[i], s[i]));
			else
				CK(hipGraphLaunch(both, s[0]));
			b[1].enqueue(b[1].ref, nullptr);  // beside them, with its own workspaces and outputs
			CK(hipDeviceSynchronize());
			const char* name[] = {"streams", "graphs", "branches"};
			for (auto& x : b) live += x.check(name[how], round);
		}
		printf("round %d\n", round);
		fflush(stdout);
	}
	if (live < 4 * 3 * 63) {  // at least half of the rows of both operators computed
		printf("only %d rows of results: the check would say little\n", live);
		return 1;
	}
	printf("ok (%d rows)\n", live);
	return 0;
}
