"""GPU: the decoder operators at the edges of what they document: pools beyond 2^31 elements,
launch hints that do not fit, outputs that overlap inputs, graphs that share a pool, a first call
inside a capture."""
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_paged_attention import DEV, check, make, run

pytestmark = pytest.mark.gpu


def test_pools_beyond_32_bits():
    """Pages at the far end of a pool of 4.5 GB: the same bits as in a small pool."""
    from qik.paged_kv import copy_pages
    from qik.rotary import rotary_store, rotary_table
    HK, page, D, N = 8, 64, 128, 34000  # 2^31 elements end at page 32768
    big = [torch.zeros(N, HK, page, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    for new, kv in (([1, 3], [900, 130]), ([200, 1], [700, 333])):
        s = make(new, kv, 16, HK, D, page, torch.bfloat16, seed=41)
        small = [s["k_pages"], s["v_pages"]]
        n, far = small[0].shape[0], N - small[0].shape[0]
        for b, p in zip(big, small):
            b[far:] = p
        want = run(s)
        t = dict(s, k_pages=big[0], v_pages=big[1], page_table=s["page_table"] + far)
        assert torch.equal(run(t), want)
        # the same new tokens stored at both
        T = sum(new)
        g = torch.Generator(device=DEV).manual_seed(42)
        q, k, v = (torch.randn(T, h, D, generator=g, device=DEV).bfloat16() for h in (16, HK, HK))
        pos = torch.arange(T, device=DEV)
        slots = torch.randperm(n * page, generator=torch.Generator().manual_seed(43))[:T].to(DEV)
        table = rotary_table(D, T)
        a = rotary_store(q, k, v, pos, table, slots, *small)
        b = rotary_store(q, k, v, pos, table, slots + far * page, *big)
        assert torch.equal(a, b) and all(torch.equal(x[far:], y) for x, y in zip(big, small))
        # pages copied from one end to the other and back
        copy_pages(*big, [(far + i, i, page) for i in range(n)])
        assert all(torch.equal(x[:n], y) for x, y in zip(big, small))
        big[0][far:] = 0
        copy_pages(*big, [(i, far + i, page) for i in range(n)])
        assert torch.equal(big[0][far:], small[0])


@pytest.mark.parametrize("new,kv", [([1, 3], [3000, 130]), ([1] * 200, [600] * 200), ([9, 20], [1500, 20]), ([300, 1], [700, 2000]),
                                    ([40] * 90, [90] * 90)])
@pytest.mark.parametrize("window", [0, 100])
def test_max_kv_only_chooses_launch_shapes(new, kv, window):
    s = make(new, kv, 8, 2, 64, 32, torch.bfloat16, seed=45)
    for max_kv in (0, 1, 500, 2 ** 62):
        check(run(s, max_kv=max_kv, window=window), s, new, kv, window=window)


def test_out_may_not_overlap_what_is_read():
    from qik.paged_attention import paged_attention
    s = make([2, 1], [40, 70], 4, 2, 64, 16, torch.bfloat16, seed=46)
    fused = torch.zeros(3, 8, 64, dtype=torch.bfloat16, device=DEV)
    fused[:, :4] = s["q"]
    want = run(s)
    t = dict(s, q=fused[:, :4])
    assert torch.equal(run(t, out=fused[:, 4:]), want)  # columns next to q's in one allocation
    with pytest.raises(ValueError, match="overlaps"):
        paged_attention(**t, out=fused[:, :4])
    with pytest.raises(ValueError, match="overlaps"):
        paged_attention(**s, out=s["q"])
    with pytest.raises(ValueError, match="overlaps"):
        paged_attention(**s, out=s["k_pages"].view(-1)[:3 * 4 * 64].view(3, 4, 64))
    with pytest.raises(ValueError, match="overlaps"):
        paged_attention(**s, out=torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV).expand(3, 4, 64))


def test_table_and_lengths_as_views():
    new, kv = [1, 5], [100, 600]
    s = make(new, kv, 4, 2, 128, 32, torch.bfloat16, seed=47)
    wide = torch.full((2, s["page_table"].shape[1] + 5), 10 ** 6, dtype=torch.int32, device=DEV)
    wide[:, 2:-3] = s["page_table"]
    lens = torch.zeros(4, dtype=torch.int32, device=DEV)
    lens[::2] = s["seq_lens"]
    t = dict(s, page_table=wide[:, 2:-3], seq_lens=lens[::2])
    assert torch.equal(run(t), run(s))


def test_graphs_of_one_pool():
    """Two captured graphs whose workspaces come from one memory pool, replayed in turn."""
    from qik.paged_attention import paged_attention
    from qik.rms_norm import fused_add_rms_norm_e4m3
    cases = [([1, 1], [9000, 700]), ([90], [4000])]
    states = [make(n, m, 8, 2, 128, 64, torch.bfloat16, seed=48 + i) for i, (n, m) in enumerate(cases)]
    w = torch.ones(1024, dtype=torch.bfloat16, device=DEV)

    def call(s):
        o = paged_attention(**s)
        return o, *fused_add_rms_norm_e4m3(o.flatten(1), o.flatten(1), w, 1e-6)[:2]
    want = [[x.clone() for x in call(s)] for s in states]
    torch.cuda.synchronize()
    graphs, got, pool = [], [], torch.cuda.graph_pool_handle()
    outs = [[torch.empty_like(x) for x in ws] for ws in want]
    for s, o in zip(states, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            for kept, x in zip(o, call(s)):
                kept.copy_(x)
    for _ in range(4):
        for g, o, ws in zip(graphs, outs, want):
            for x in o:
                x.zero_()
            g.replay()
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(o, ws))


FIRST = """
import torch
from qik import _lib as L
from qik.paged_attention import paged_attention
d = dict(device="cuda")
q, k, v = (torch.randn(n, 2, m, 64, **d).bfloat16() for n, m in ((1, 1), (4, 16), (4, 16)))
i32 = dict(dtype=torch.int32, **d)
args = (q.view(1, 2, 64), k, v, torch.tensor([[2, 0]], **i32), torch.tensor([20], **i32), torch.tensor([0, 1], **i32), 1)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = paged_attention(*args)
word = L.status_word(torch.device("cuda", 0))
assert L.device_status() == 0
word.fill_(7)
g.replay()
assert L.device_status() == 7, "the graph writes the status word"
word.zero_()
assert torch.equal(out, paged_attention(*args)) and L.device_status() == 0
"""


def test_first_call_inside_a_capture():
    """A new process whose first call is captured: its status word is made outside of the graph."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-image-kernel_b200")
    done = subprocess.run([sys.executable, "-c", FIRST], env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
