"""GPU: paged attention over caches in which infinities and NaN have spread: what comes out, and that
forming rows again neither runs into the limit of the other waits nor takes long where it changes nothing."""
import pytest
import torch

from test_gpu_paged_attention import DEV, check, exact, make

pytestmark = pytest.mark.gpu


def timed(s, **kw):
    """(out, device milliseconds); no wait may have given up."""
    from qik import _lib as L
    from qik.paged_attention import paged_attention
    dev = torch.device(DEV, 0)
    L.status_word(dev).zero_()
    paged_attention(**s, **kw)
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    out = paged_attention(**s, **kw)
    b.record()
    torch.cuda.synchronize()
    assert L.device_status(dev) == 0
    return out, a.elapsed_time(b)


def places(s, i, t):
    t = torch.as_tensor(t)
    return s["page_table"][i].cpu().long()[t // 64].to(DEV), (t % 64).to(DEV)


@pytest.mark.parametrize("new,kv,heads,kv_heads,dim", [([8001], [8001], 8, 8, 128), ([20000], [20000], 4, 1, 64), ([8] * 40, [6000] * 40, 16, 4, 128)])
def test_a_cache_of_nan_takes_no_longer_than_rows_do(new, kv, heads, kv_heads, dim):
    """Every row that sees NaN sees it at its own place, so it is not formed again key by key; with NaN
    from the middle on, the rows before it in its own block are.  (The limit where there are none, 100
    times the finite call, is a tenth of what forming all rows again would take.)"""
    s = make(new, kv, heads, kv_heads, dim, 64, torch.bfloat16, seed=3)
    want, finite = timed(s)
    for from_ in (0, kv[0] // 2):
        t = dict(s, v_pages=s["v_pages"].clone())
        for i, m in enumerate(kv):
            page, at = places(s, i, torch.arange(from_, m))
            t["v_pages"][page, :, at] = float("nan")
        got, ms = timed(t)
        at = 0
        for n, m in zip(new, kv):
            blind = max(0, from_ - (m - n))  # rows before the first NaN
            assert got[at + blind:at + n].isnan().all()
            assert (got[at:at + blind].float() - want[at:at + blind].float()).abs().max() < 0.02 if blind else True
            at += n
        assert from_ or ms < max(100 * finite, 10.0), (ms, finite)


def test_rows_before_an_infinity_in_a_long_prompt():
    """1.3 million tokens, infinity in V at the last one: the rows of its block that do not see it
    are formed again over all their keys, which takes longer than a wait may."""
    T = 1_300_000
    s = make([T], [T], 1, 1, 64, 64, torch.bfloat16, seed=4)
    want, _ = timed(s)
    page, at = places(s, 0, T - 1)
    s["v_pages"][page, 0, at, 3] = float("inf")
    from qik import _lib as L
    from qik.paged_attention import paged_attention
    got = paged_attention(**s)
    torch.cuda.synchronize()
    assert L.device_status(torch.device(DEV, 0)) == 0
    assert got[-1, 0, 3] == float("inf") and got.isfinite().sum() == got.numel() - 1
    rest = torch.arange(64, device=DEV) != 3
    assert torch.equal(got[..., rest], want[..., rest])
    # 1e6 values of deviation 1 under nearly equal weights: outputs of about 1e-3, p rounded by 2^-8 in one of them
    off = (got[:-1, 0, 3].double() - want[:-1, 0, 3].double()).abs()
    few = torch.arange(T - 1, device=DEV) < T - 256
    assert (off[few] == 0).all() and off[~few].max() < 1e-3 * 2.0 ** -6


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("new,kv,window,sinks", [([9, 3], [300, 64], 0, 0), ([7], [900], 200, 5), ([200, 90], [700, 90], 0, 0), ([300], [1500], 500, 3)])
def test_columns_are_formed_again_one_by_one(new, kv, window, sinks, dtype, dim):
    """A row that sees NaN in one column and not the infinity in another: the first stays NaN, the
    second is exact."""
    s = make(new, kv, 4, 2, dim, 64, dtype, seed=5)
    clean = dict(s, v_pages=s["v_pages"].clone())
    nans, infs = [], []
    for i, (n, m) in enumerate(zip(new, kv)):
        for t, col, value, told in ((m - n, 7, float("nan"), nans), (m - 1, 8, float("inf"), infs), (m - 1, dim - 1, -float("inf"), infs)):
            page, at = places(s, i, t)
            s["v_pages"][page, :, at, col] = value
            told.append((i, t, col, value))
    got, _ = timed(s, window=window, sinks=sinks)
    want, _ = exact(clean, new, kv, window=window, sinks=sinks)
    start = 0
    for i, n in enumerate(new):
        for told in (nans, infs):
            for seq, t, col, value in told:
                for j in range(n if seq == i else 0):
                    last = kv[i] - n + j
                    if t <= last and (not window or t > last - window or t < sinks):
                        x = got[start + j, :, col]
                        assert x.isnan().all() if value != value else (x == value).all()
                        got[start + j, :, col] = want[start + j, :, col].to(dtype)
        start += n
    check(got, clean, new, kv, window=window, sinks=sinks)
