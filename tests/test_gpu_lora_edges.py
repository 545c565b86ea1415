"""The per-row adapters' projection at the edges of its domain: the smallest depth and width past 64 rows, the
largest depth, the widest row (tests/test_gpu_batch_ops.py has the sizes between)."""
import pytest

from test_gpu_batch_ops import LoraBatch, dev, host, ops  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k,ranks,rows", [
    (65, 16, 16, [1, 64], [0, 1, -1]),
    (66, 8192, 48, [3], [0, -1]),
    (512, 32, 32768, [64, 1], [0, 1]),
    (64, 16, 32768, [64, 5], [1, 0, -1]),
    (1, 8192, 16, [64], [0]),
    (1, 8192, 32768, [33], [0]),
])
def test_lora_at_the_edges(m, n, k, ranks, rows, ops, dev, host):  # noqa: F811
    print(f"case lora edge {m}x{n}x{k} {ranks}", flush=True)
    b = LoraBatch(m + n + k, m, n, k, ranks, rows)
    b.check(host, b.run(ops, dev))


def test_lora_extreme_codes(ops, dev, host):  # noqa: F811
    """Every product at its largest: codes of -128 in the inputs, weights and adapters, at the largest depth."""
    b = LoraBatch(1, 3, 16, 32768, [64, 64], [0, -1, 1])
    b.a[...] = -128
    b.w[...] = -128
    for i, (a, uf, lb, df) in enumerate(b.adapters):
        a[...] = -128 if i == 0 else 127
        lb[...] = -128
        df[:, 2] = range(-8, 8)
    print("case lora extreme codes", flush=True)
    b.check(host, b.run(ops, dev))
