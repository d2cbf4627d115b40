"""GPU: page copies in pools whose pages hold tokens of heads or heads of tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pools(layers, N, H, page, D, dtype, pad=0):
    """Two pools [layers, N, H, page, D] that lie as [layers, N, page, H, D], `pad` heads apart."""
    g = torch.Generator(device=DEV).manual_seed(7)
    return [torch.randn(layers, N, page, H + pad, D, generator=g, device=DEV).to(dtype)[..., :H, :].transpose(2, 3) for _ in range(2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layers,H,page,D", [(3, 4, 16, 64), (1, 8, 128, 128), (2, 1, 32, 64), (2, 3, 64, 72)])
def test_heads_of_tokens(layers, H, page, D, dtype):
    from qik.paged_kv import copy_pages
    k, v = pools(layers, 12, H, page, D, dtype)
    moves = [(0, 5, page), (3, 7, 1), (0, 2, page // 2 + 1), (8, 9, 0), (11, 10, page - 1)]
    want = [k.clone(), v.clone()]
    for p, w in zip((k, v), want):
        for a, b, t in moves:
            w[:, b, :, :t] = p[:, a, :, :t]
    copy_pages(k, v, moves)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    w = k[0].clone()
    w[1, :, :3] = w[4, :, :3]
    copy_pages(k[0], v[0], [(4, 1, 3)])
    assert torch.equal(k[0], w)


def test_a_fork_of_such_a_pool_is_attended_to():
    """What rotary_store and paged_attention take can be copied too: the same outputs from the copied page."""
    from qik.paged_kv import copy_pages
    from test_gpu_paged_attention import make, run
    s = make([1, 3], [90, 100], 4, 2, 64, 64, torch.bfloat16, seed=8)
    t = dict(s)
    for name in ("k_pages", "v_pages"):
        t[name] = torch.empty_like(s[name].transpose(1, 2).contiguous()).transpose(1, 2)
        t[name].copy_(s[name])
    want = run(s)
    used = {x for row, kv in zip(s["page_table"].tolist(), (90, 100)) for x in row[:-(-kv // 64)]}
    to = next(i for i in range(s["k_pages"].shape[0]) if i not in used)
    old = int(s["page_table"][1, 1])
    copy_pages(t["k_pages"], t["v_pages"], [(old, to, 36)])
    t["k_pages"][old], t["v_pages"][old] = 0, 0
    t["page_table"] = t["page_table"].clone()
    t["page_table"][1, 1] = to
    assert torch.equal(run(t), want)


def test_other_strides_are_refused():
    from qik.paged_kv import copy_pages
    k, v = pools(2, 4, 3, 16, 64, torch.bfloat16, pad=1)
    plain = torch.zeros(2, 4, 3, 16, 64, dtype=torch.bfloat16, device=DEV)
    wide = torch.zeros(2, 4, 3, 16, 128, dtype=torch.bfloat16, device=DEV)[..., :64]
    near, _ = pools(2, 4, 3, 16, 64, torch.bfloat16)
    for a, b in ((k, v), (plain, near), (near, plain), (wide, wide), (plain, wide)):
        before = a.clone()
        with pytest.raises(ValueError, match="contiguous"):
            copy_pages(a, b, [(0, 1, 1)])
        assert torch.equal(a, before)
