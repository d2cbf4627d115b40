"""GPU: the status word keeps the graver report: an index outside its tensor does not replace a wait
that gave up, which is reported whatever the word held."""
import pytest
import torch

from test_gpu_paged_attention import DEV, make

pytestmark = pytest.mark.gpu


def bad_calls():
    from qik.paged_attention import paged_attention
    from qik.rotary import apply_rotary, rotary_store, rotary_table
    for new in ([1, 1], [90, 100]):
        for what in ("page", "length"):
            s = make(new, [300, 400], 4, 2, 64, 64, torch.bfloat16, seed=81)
            s["page_table" if what == "page" else "seq_lens"].view(-1)[1] = 10 ** 6
            yield lambda s=s: paged_attention(**s)
    x = torch.randn(3, 2, 64, device=DEV).bfloat16()
    table, pos = rotary_table(64, 8), torch.tensor([0, 9, 1], device=DEV)
    pages = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    yield lambda: apply_rotary(x, x, pos, table)
    yield lambda: rotary_store(x, x, x, pos % 8, table, torch.tensor([1, 2, 32], device=DEV), pages, pages.clone())


@pytest.mark.parametrize("at", range(6))
def test_a_bad_index_does_not_replace_a_timeout(at):
    from qik import _lib as L
    dev = torch.device(DEV, 0)
    call = list(bad_calls())[at]
    word = L.status_word(dev)
    for before, after in ((L.STATUS_OK, L.STATUS_BAD_INDEX), (L.STATUS_TIMEOUT, L.STATUS_TIMEOUT), (L.STATUS_BAD_INDEX, L.STATUS_BAD_INDEX)):
        word[0] = before
        call()
        torch.cuda.synchronize()
        assert L.device_status(dev) == after
    word.zero_()
