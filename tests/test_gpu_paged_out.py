"""GPU: which outputs paged attention takes beside what it reads: views of one allocation are taken
where no element is shared, and refused otherwise, before anything is launched."""
import pytest
import torch

from test_gpu_paged_attention import DEV, make, run

pytestmark = pytest.mark.gpu
T, H, D = 5, 4, 64
NEW, KV = [2, 3], [40, 70]


def views():
    """(name, q's view, out's view, whether they are apart) of one allocation."""
    def rows(n):
        return torch.zeros(T, n, D, dtype=torch.bfloat16, device=DEV)
    x = rows(8)
    yield "next to each other", x[:, :4], x[:, 4:], True
    yield "the other way round", x[:, 4:], x[:, :4], True
    for k in (1, 2, 3):
        yield f"{k} heads on", x[:, :4], x[:, k:k + 4], False
    yield "half a head on", x[:, :4], x.view(T, 8 * D)[:, 32:32 + 4 * D].unflatten(1, (4, D)), False
    x = rows(12)
    yield "a gap between", x[:, :4], x[:, 7:11], True
    yield "the same", x[:, 2:6], x[:, 2:6], False
    yield "one head shared", x[:, 5:9], x[:, 2:6], False
    x = torch.zeros(T, H, 3, D, dtype=torch.bfloat16, device=DEV)
    yield "heads in turn", x[:, :, 0], x[:, :, 2], True
    yield "heads in turn, shifted", x[:, :, 0], x.view(T, H * 3 * D)[:, 8:].as_strided((T, H, D), (H * 3 * D, 3 * D, 1)), False
    x = torch.zeros(H, 2, T, D, dtype=torch.bfloat16, device=DEV)
    yield "heads outside", x[:, 0].transpose(0, 1), x[:, 1].transpose(0, 1), True
    x = torch.zeros(2 * T, H, D, dtype=torch.bfloat16, device=DEV)
    yield "tokens behind", x[:T], x[T:], True
    yield "tokens in turn", x[::2], x[1::2], True
    yield "one token on", x[:T], x[1:T + 1], False
    yield "tokens in turn and not", x[::2], x[T:], False


@pytest.mark.parametrize("at", range(16))
def test_out_and_q_in_one_allocation(at):
    from qik.paged_attention import paged_attention
    name, q, out, apart = list(views())[at]
    s = make(NEW, KV, H, 2, D, 16, torch.bfloat16, seed=71)
    want = run(s)
    q.copy_(s["q"])
    t = dict(s, q=q)
    if apart:
        assert torch.equal(run(t, out=out), want) and torch.equal(q, s["q"]), name
    else:
        with pytest.raises(ValueError, match="overlaps"):
            paged_attention(**t, out=out)


def test_there_is_a_case_for_each_view():
    assert len(list(views())) == 16


def test_out_that_overlaps_itself_or_the_pages():
    from qik.paged_attention import paged_attention
    s = make(NEW, KV, H, 2, D, 16, torch.bfloat16, seed=72)
    flat = torch.zeros(4096, dtype=torch.bfloat16, device=DEV)
    for strides in ((D, D, 1), (H * D, 32, 1), (H * D - 8, D, 1), (8, T * D, 1)):
        with pytest.raises(ValueError, match="overlaps"):
            paged_attention(**s, out=flat.as_strided((T, H, D), strides))
    both = torch.zeros(s["k_pages"].shape[0], 2, 2, 16, D, dtype=torch.bfloat16, device=DEV)  # pages of k and v in turn
    both[:, 0], both[:, 1] = s["k_pages"], s["v_pages"]
    t = dict(s, k_pages=both[:, 0], v_pages=both[:, 1])
    want = run(s)
    assert torch.equal(run(t), want)
    for pages in (both[:, 0], both[:, 1]):
        with pytest.raises(ValueError, match="overlaps"):
            paged_attention(**t, out=pages[:T].reshape(T, -1, D)[:, :H] if pages.is_contiguous() else pages[:T, 0, :H])
    own = dict(s, k_pages=torch.cat((s["k_pages"].flatten(), flat[:T * H * D])))
    own["k_pages"], out = own["k_pages"][:s["k_pages"].numel()].view_as(s["k_pages"]), own["k_pages"][s["k_pages"].numel():].view(T, H, D)
    assert torch.equal(run(own, out=out), want)
