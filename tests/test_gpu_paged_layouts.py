"""GPU: paged attention and the rotary store over pools of every stride that they take, and groups of up
to 64 query heads a key head, against the definition in 64 bits (bounds: test_gpu_paged_attention)."""
import pytest
import torch

from test_gpu_paged_attention import DEV, check, make, run

pytestmark = pytest.mark.gpu


def lay(name, shape, dtype, fill=float("nan")):
    """An empty pool [pages, heads, page, D] laid out as `name` says; what lies between is `fill`."""
    N, H, P, D = shape
    def buf(*s):
        return torch.full(s, fill, dtype=dtype, device=DEV)
    if name == "tokens outside heads":
        return buf(N, P, H, D).permute(0, 2, 1, 3)
    if name == "heads outside":
        return buf(H, N, P, D).permute(1, 0, 2, 3)
    if name == "padded columns":
        return buf(N, H, P, D + 8)[..., :D]
    if name == "padded everything":
        return buf(2 * N, H + 3, P + 5, D + 24)[::2, 1:H + 1, 2:P + 2, 8:D + 8]
    if name == "half of each page":
        return buf(N, 2, H, P, D)[:, 1]
    if name == "tokens outside pages' heads, wide":
        return buf(N, P, H, 2, D)[..., 0, :].permute(0, 2, 1, 3)
    return buf(N, H, P, D)


LAYOUTS = [("tokens outside heads", "tokens outside heads"), ("heads outside", "plain"), ("plain", "padded columns"),
           ("padded everything", "half of each page"), ("tokens outside pages' heads, wide", "heads outside")]
CALLS = [([1, 1, 1], [5, 900, 4000], {}), ([3, 9, 16], [300, 64, 2000], {}), ([200, 1, 70], [700, 1300, 70], {}),
         ([200, 90], [200, 700], dict(causal=False)), ([9, 2], [3000, 77], dict(window=100, sinks=5)),
         ([150, 300], [2500, 300], dict(window=64, sinks=130)), ([300], [9000], {})]


@pytest.mark.parametrize("dtype,dim,page", [(torch.bfloat16, 128, 64), (torch.float16, 64, 16), (torch.bfloat16, 64, 256), (torch.float16, 128, 32)])
@pytest.mark.parametrize("call", range(len(CALLS)))
@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
def test_any_strides_of_the_pools(layout, call, dtype, dim, page):
    new, kv, kw = CALLS[call]
    s = make(new, kv, 8, 2, dim, page, dtype, seed=90 + call)
    t = dict(s)
    for name, how in zip(("k_pages", "v_pages"), LAYOUTS[layout]):
        t[name] = lay(how, s[name].shape, dtype)
        t[name].copy_(s[name])
    got = run(t, **kw)
    assert torch.equal(got, run(s, **kw))
    if layout == 0:
        check(got, s, new, kv, **kw)


@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
@pytest.mark.parametrize("new,kv,window", [([9, 4], [200, 1000], 0), ([13], [300], 30), ([200, 90], [200, 700], 0), ([300], [900], 64)])
def test_rows_formed_again_from_any_strides(layout, new, kv, window):
    """Infinities and NaN that some rows do not see, in pools of other strides."""
    s = make(new, kv, 8, 2, 64, 32, torch.bfloat16, seed=95)
    for i, (n, m) in enumerate(zip(new, kv)):
        for t, col, value in ((m - 1, 5, float("nan")), (m - 1 - n // 2, 40, float("inf")), (max(0, m - n - window), 41, -float("inf"))):
            s["v_pages"][s["page_table"][i, t // 32].long(), :, t % 32, col] = value
    t = dict(s)
    for name, how in zip(("k_pages", "v_pages"), LAYOUTS[layout]):
        t[name] = lay(how, s[name].shape, torch.bfloat16)
        t[name].copy_(s[name])
    got, want = run(t, window=window), run(s, window=window)
    assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0)) and got.isnan().any() and got.isinf().any()


@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
@pytest.mark.parametrize("D,rot,interleaved,HK", [(128, 128, False, 3), (64, 32, True, 1), (256, 96, False, 2)])
def test_rotary_store_into_any_strides(layout, D, rot, interleaved, HK):
    """The same bits at the same places, nothing between them."""
    from qik.rotary import rotary_store, rotary_table
    g = torch.Generator(device=DEV).manual_seed(96)
    T, page, pages = 77, 32, 9
    q, k, v = (torch.randn(T, h, D, generator=g, device=DEV).bfloat16() for h in (4, HK, HK))
    table, pos = rotary_table(rot, 500), torch.randint(0, 500, (T,), generator=g, device=DEV)
    slots = torch.randperm(page * pages, generator=g, device=DEV)[:T]
    slots[5] = -1
    plain = [torch.full((pages, HK, page, D), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    pools = [lay(how, (pages, HK, page, D), torch.bfloat16, fill=3.0) for how in LAYOUTS[layout]]
    a, b = (rotary_store(q, k, v, pos, table, slots, *p, interleaved=interleaved) for p in (plain, pools))
    assert torch.equal(a, b)
    for x, y in zip(plain, pools):
        assert torch.equal(x, y)
        whole = torch.as_strided(y, (y.untyped_storage().nbytes() // 2,), (1,), 0)
        assert (whole != 3).sum() == (y != 3).sum()


GROUPS = [9, 12, 16, 17, 31, 33, 43, 48, 63, 64]


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("new,kv,kw", [([1, 1], [300, 2000], {}), ([1], [30], {}), ([2, 1, 3], [700, 64, 3], {}), ([7, 40], [50, 1200], {}),
                                       ([65, 1], [65, 400], dict(causal=False)), ([5, 33], [900, 500], dict(window=70, sinks=3))])
def test_wide_groups(new, kv, kw, group, dtype, dim):
    """9 to 64 query heads a key head: a few tokens a query tile, rows of the tile that hold none."""
    HK = 2 if group < 40 else 1
    s = make(new, kv, group * HK, HK, dim, 64, dtype, seed=group, strided=group % 2 == 1)
    check(run(s, **kw), s, new, kv, **kw)


def test_more_than_64_heads_a_key_head_are_refused():
    from qik import _lib as L
    from qik.paged_attention import paged_attention
    s = make([1], [30], 65, 1, 64, 64, torch.bfloat16, seed=1)
    with pytest.raises(L.QikError, match="65 query heads"):
        paged_attention(**s)
