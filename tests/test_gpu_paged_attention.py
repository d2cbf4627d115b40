"""GPU: attention over a paged cache (qik.paged_attention) against the definition in 64 bits.

The bound on |out - exact| is element by element, from the roundings the kernels make: p is
rounded to the tensors' type (half a step, eps / 2, of each p v term), the result once more;
2^x costs at most 1e-4 relative (the cubic on the FMA pipe 7.5e-5, ex2.approx 2^-22), and the
fp32 scores and sums stay under that.  In fp16 a p below 2^-14 is rounded by up to 2^-25.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(new, kv, heads, kv_heads, dim, page, dtype, seed=0, spare=3, strided=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T = sum(new)
    need = [-(-n // page) for n in kv]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    W = max(need + [1]) + 1
    table = torch.full((len(new), W), 10 ** 6, dtype=torch.int32)  # unused entries are never followed
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = torch.tensor(order[at:at + m], dtype=torch.int32)
        at += m
    q = torch.randn(T, heads, dim, generator=g, device=DEV).to(dtype)
    if strided:
        qkv = torch.randn(T, (heads + 2) * dim, generator=g, device=DEV).to(dtype)
        q = qkv[:, dim:(heads + 1) * dim].unflatten(1, (heads, dim))
    k, v = (torch.randn(pages, kv_heads, page, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    return dict(q=q, k_pages=k, v_pages=v, page_table=table.to(DEV),
                seq_lens=torch.tensor(kv, dtype=torch.int32, device=DEV), query_starts=starts.to(DEV),
                max_new=max(new + [0]))


def exact(s, new, kv, causal=True, window=0, sinks=0, scale=None):
    """(out, sum p |v| / sum p) of every new token in 64 bits."""
    page = s["k_pages"].shape[2]
    HK, H, D = s["k_pages"].shape[1], s["q"].shape[1], s["q"].shape[2]
    scale = D ** -0.5 if scale is None else scale
    out, mass = [], []
    table = s["page_table"].cpu().long()
    at = 0
    for i, (n, m) in enumerate(zip(new, kv)):
        t = torch.arange(m)
        where = (table[i][t // page].to(DEV), (t % page).to(DEV))
        k, v = (p[where[0], :, where[1]].double().repeat_interleave(H // HK, 1) for p in (s["k_pages"], s["v_pages"]))
        q = s["q"][at:at + n].double()
        t = t.to(DEV)
        last = m - n + torch.arange(n, device=DEV) if causal else torch.full((n,), m - 1, device=DEV)
        seen = t[None] <= last[:, None]
        if window:
            seen &= (t[None] > last[:, None] - window) | (t[None] < sinks)
        a = torch.einsum("nhd,mhd->hnm", q, k) * scale
        a = a.masked_fill(~seen, -math.inf)
        top = a.amax(-1, keepdim=True) if m else a.new_zeros(H, n, 1)
        p = torch.where(seen, torch.exp(a - torch.where(top == -math.inf, 0.0, top)), 0.0)
        total = p.sum(-1)[..., None]
        p = torch.where(total > 0, p / total, 0.0)
        v0 = torch.where((seen.any(0) if n else t < 0)[:, None, None], v, 0.0)  # 0 x NaN is no contribution
        out.append(torch.einsum("hnm,mhd->nhd", p, v0))
        mass.append(torch.einsum("hnm,mhd->nhd", p, v0.abs()))
        at += n
    return torch.cat(out), torch.cat(mass)


def check(got, s, new, kv, **kw):
    want, mass = exact(s, new, kv, **kw)
    half = torch.finfo(got.dtype).eps / 2
    tiny = max(kv + [1]) * 2.0 ** -25 * 8 if got.dtype == torch.float16 else 0.0
    bound = (half + 1.5e-4) * mass + half * want.abs() + tiny + 1e-6
    T = want.shape[0]
    off = (got[:T].double() - want).abs()
    assert torch.isfinite(got[:T]).all()
    worst = (off / bound).max().item() if T else 0.0
    assert worst <= 1.0, f"{worst} of the bound"


def run(s, **kw):
    from qik import _lib as L
    from qik.paged_attention import paged_attention
    L.status_word(torch.device(DEV, 0)).zero_()
    got = paged_attention(**s, **kw)
    torch.cuda.synchronize()
    assert L.device_status(torch.device(DEV, 0)) == 0
    return got


SMALL = [  # new, kv, heads, kv heads
    ([1], [1], 1, 1), ([1], [300], 32, 8), ([1, 1, 1], [17, 64, 65], 8, 8), ([1] * 5, [1, 5000, 63, 129, 2047], 7, 1),
    ([3, 1, 16], [3, 700, 1000], 4, 1), ([2, 5], [513, 4000], 16, 4), ([13], [2000], 5, 1), ([1], [40000], 8, 1),
    ([1] * 70, list(range(5, 705, 10)), 4, 2), ([4, 0, 1], [100, 30, 0], 4, 2), ([0, 2], [0, 600], 2, 2),
    ([1] * 300, [600] * 300, 2, 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("case", range(len(SMALL)))
def test_few_rows(case, dim, dtype):
    new, kv, H, HK = SMALL[case]
    s = make(new, kv, H, HK, dim, (16, 64, 32, 128, 256)[case % 5], dtype, seed=case)
    check(run(s), s, new, kv)
    check(run(s, max_kv=max(kv)), s, new, kv)


LARGE = [([65], [65], 1, 1), ([128], [128], 2, 2), ([100], [1000], 8, 2), ([257, 64, 300], [257, 640, 1300], 3, 1),
         ([130, 33], [4130, 2033], 28, 4), ([1, 500, 1], [900, 500, 3000], 8, 1), ([700], [700], 5, 5),
         ([20, 300], [5, 290], 8, 2), ([513], [9000], 4, 4)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("case", range(len(LARGE)))
def test_many_rows(case, dim, dtype):
    """Chunks, prompts and mixed batches; more new tokens than the cache holds (rows that see
    nothing are zeros)."""
    new, kv, H, HK = LARGE[case]
    s = make(new, kv, H, HK, dim, (64, 16, 128, 32, 512)[case % 5], dtype, seed=50 + case, strided=case % 2 == 1)
    check(run(s), s, new, kv)
    check(run(s, causal=False), s, new, kv, causal=False)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (100, 0), (128, 1), (1000, 37), (1024, 200), (5000, 4), (64, 10000)])
@pytest.mark.parametrize("new,kv", [([1, 1, 1], [5, 900, 4000]), ([9, 2], [3000, 77]), ([200, 1, 70], [2500, 1300, 70])])
def test_window_and_sinks(new, kv, window, sinks, dtype, dim):
    s = make(new, kv, 8, 2, dim, 32, dtype, seed=window)
    check(run(s, window=window, sinks=sinks), s, new, kv, window=window, sinks=sinks)


@pytest.mark.parametrize("new,kv", [([1, 1], [70, 1000]), ([5, 3], [333, 64]), ([150, 90], [150, 1000])])
@pytest.mark.parametrize("window", [0, 40])
def test_unseen_places_hold_nan(new, kv, window):
    """NaN and infinities behind the last token, in unused pages and before the window."""
    s = make(new, kv, 8, 2, 128, 64, torch.bfloat16, seed=7)
    want, _ = exact(s, new, kv, window=window, sinks=3 if window else 0)
    used = torch.zeros(s["k_pages"].shape[0], 64, dtype=torch.bool, device=DEV)
    for i, (n, m) in enumerate(zip(new, kv)):
        t = torch.arange(m)
        seen = (t > m - n - window) | (t < 3) if window else t >= 0
        used[s["page_table"][i].cpu().long()[t // 64][seen].to(DEV), (t % 64)[seen].to(DEV)] = True
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device=DEV, dtype=torch.bfloat16)
    for name in ("k_pages", "v_pages"):
        p = s[name]
        junk = bad[torch.arange(p.numel(), device=DEV) % 3].view_as(p)
        s[name] = torch.where(used[:, None, :, None], p, junk)
    check(run(s, window=window, sinks=3 if window else 0), s, new, kv, window=window, sinks=3 if window else 0)


def test_out_strides_and_rows_behind_the_last():
    new, kv = [3, 80], [100, 400]
    s = make(new, kv, 4, 2, 128, 64, torch.bfloat16, seed=9)
    s["q"] = torch.cat((s["q"], torch.randn(11, 4, 128, device=DEV).bfloat16()))
    wide = torch.full((94, 6, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    out = run(s, out=wide[:, 1:5])
    check(out, s, new, kv)
    assert (wide[83:] == 7).all() and (wide[:, 0] == 7).all() and (wide[:, 5] == 7).all()


def test_scale_and_large_scores():
    """Scores of several hundred: the running maximum moves by far more than the lazy rescale's 2^8."""
    for new, kv in (([1, 2], [3000, 500]), ([200], [1500])):
        s = make(new, kv, 4, 2, 128, 32, torch.bfloat16, seed=11)
        s["q"] = s["q"] * 6
        check(run(s, sm_scale=0.7), s, new, kv, scale=0.7)


def test_captured_graph_follows_the_lengths():
    from qik.paged_attention import paged_attention
    new = [1, 1, 1]
    s = make(new, [3000, 100, 900], 8, 2, 128, 64, torch.bfloat16, seed=13)
    out = torch.zeros(3, 8, 128, dtype=torch.bfloat16, device=DEV)
    paged_attention(**s, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged_attention(**s, out=out)
    for kv in ([3000, 100, 900], [1, 64, 65], [2999, 0, 3]):
        s["seq_lens"].copy_(torch.tensor(kv, dtype=torch.int32))
        out.fill_(5)
        g.replay()
        torch.cuda.synchronize()
        check(out, s, new, kv)


def test_two_streams_at_once():
    """Calls in flight on two streams have workspaces of their own."""
    from qik.paged_attention import paged_attention
    cases = [([1] * 4, [9000, 50, 4000, 700]), ([130], [6000])]
    states = [make(n, m, 8, 2, 128, 64, torch.bfloat16, seed=20 + i) for i, (n, m) in enumerate(cases)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i] = paged_attention(**states[i])
    torch.cuda.synchronize()
    for (n, m), s, o in zip(cases, states, outs):
        check(o, s, n, m)


def test_same_bits_every_time():
    for new, kv in (([1, 1], [20000, 3000]), ([100, 4], [9000, 100])):
        s = make(new, kv, 8, 2, 128, 64, torch.bfloat16, seed=30)
        first = run(s)
        for _ in range(5):
            assert torch.equal(first, run(s))


def test_bad_lengths_and_pages_are_reported():
    """A page outside the pool reads zeros, a length outside the table is cut: nothing else of
    the memory is touched, and the status word says so."""
    from qik import _lib as L
    from qik.paged_attention import paged_attention
    dev = torch.device(DEV, 0)
    for new, kv in (([1, 1], [500, 900]), ([100, 90], [500, 900])):
        for what in ("page", "negative page", "length"):
            s = make(new, kv, 4, 2, 128, 64, torch.bfloat16, seed=31)
            if what == "length":
                s["seq_lens"][0] = 10 ** 6
            else:
                s["page_table"][0, 2] = 10 ** 6 if what == "page" else -5
            L.status_word(dev).zero_()
            out = paged_attention(**s)
            torch.cuda.synchronize()
            assert L.device_status(dev) == L.STATUS_BAD_INDEX
            L.status_word(dev).zero_()
            want, _ = exact(make(new, kv, 4, 2, 128, 64, torch.bfloat16, seed=31), new, kv)
            n = new[0]
            assert (out[n:].double() - want[n:]).abs().max() < 0.05  # the other sequence is whole


def test_empty_calls():
    from qik.paged_attention import paged_attention
    k = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    out = paged_attention(torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=DEV), k, k, torch.zeros(0, 0, **i32),
                          torch.zeros(0, **i32), torch.zeros(1, **i32), 0)
    assert out.shape == (0, 4, 64)
    q = torch.ones(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    out = paged_attention(q, k, k, torch.zeros(2, 0, **i32), torch.zeros(2, **i32), torch.tensor([0, 1, 2], **i32), 1)
    torch.cuda.synchronize()
    assert (out == 0).all()


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("new,kv,window", [([9, 1, 4], [200, 64, 1000], 0), ([5], [700], 30), ([13], [40], 0), ([60], [130], 20),
                                           ([200, 90], [200, 700], 0), ([300], [900], 64), ([129, 7], [2000, 9], 0)])
def test_infinities_in_keys_that_some_rows_see(new, kv, window, dtype, dim):
    """V with infinities and NaN at new tokens and at a window's edge: rows that do not see the
    token are exact, rows that do have what the formula gives in each column."""
    s = make(new, kv, 8, 2, dim, 32, dtype, seed=17)
    odd = []
    for i, (n, m) in enumerate(zip(new, kv)):
        for back, value, col in ((0, float("nan"), 3), (n // 2, float("inf"), 7), (n - 1, -float("inf"), dim - 1),
                                 (min(m - 1, window + n // 3), float("inf"), 20)):
            t = m - 1 - back
            s["v_pages"][s["page_table"][i, t // 32].long(), 1, t % 32, col] = value
            odd.append((i, t, col))
    got = run(s, window=window)
    finite = dict(s, v_pages=torch.where(s["v_pages"].isfinite(), s["v_pages"], torch.zeros_like(s["v_pages"])))
    want, mass = exact(finite, new, kv, window=window)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    touched = torch.zeros(got.shape, dtype=torch.bool, device=DEV)
    for i, t, col in set(odd):
        value = s["v_pages"][s["page_table"][i, t // 32].long(), 1, t % 32, col].double()
        for j in range(new[i]):
            last = kv[i] - new[i] + j
            if t <= last and (not window or t > last - window):
                want[starts[i] + j, 4:, col] += value  # p is positive
                touched[starts[i] + j, 4:, col] = True
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()].double(), want[want.isinf()])
    half = torch.finfo(dtype).eps / 2
    bound = (half + 1.5e-4) * mass + half * want.abs() + (max(kv) * 2.0 ** -22 if dtype == torch.float16 else 0) + 1e-6
    assert ((got.double() - want).abs()[~touched] <= bound[~touched]).all()
    assert touched.any() and not touched.all()
