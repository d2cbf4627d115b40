"""GPU: paged attention whose CTAs walk ranges of many units, against the definition in 64 bits:
units without keys in runs behind units with keys, more sequences than a CTA has threads.

The bound is that of test_gpu_paged_attention.
"""
import pytest
import torch

from test_gpu_paged_attention import check, make, run

pytestmark = pytest.mark.gpu

# (new, kv, heads, kv heads, keywords): sequences and row blocks that see no key, next to long ones
RUNS = [([80] * 64, [2000, 0] * 32, 8, 8, {}),
        ([80] * 64, [2000, 0] * 32, 8, 8, dict(causal=False)),
        ([100, 70, 66, 300, 90] * 12, [3000, 0, 0, 10, 0] * 12, 6, 6, dict(causal=False)),
        ([100, 70, 66, 300, 90] * 12, [3000, 0, 0, 10, 0] * 12, 6, 6, dict(window=900, sinks=140)),
        ([2000, 65] * 10, [10, 1100] * 10, 8, 4, {}),
        ([2000, 65] * 10, [10, 1100] * 10, 8, 4, dict(window=600, sinks=9)),
        ([2500, 100] * 6, [100, 2000] * 6, 6, 6, dict(window=50)),
        ([65, 66, 70, 90, 1] * 140, [300, 0, 0, 0, 0] * 140, 1, 1, {}),
        ([3, 200, 40] * 250, [50 * i % 900 for i in range(750)], 2, 1, {})]


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("case", range(len(RUNS)))
def test_units_without_keys(case, dtype, dim):
    """Rows that see no key are zeros, wherever they stand among rows that do."""
    new, kv, H, HK, kw = RUNS[case]
    s = make(new, kv, H, HK, dim, (64, 32, 128)[case % 3], dtype, seed=60 + case)
    check(run(s, **kw), s, new, kv, **kw)
