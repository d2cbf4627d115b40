"""CPU: the paged cache's host logic, the refusals of the decoder operators, the rotary tables."""
import ctypes
import math
import random
import struct

import pytest
import torch

# The argument structs of include/qik.h, in its order (native alignment):
# qik_rotary_args: q k v q_out k_out v_out positions slots cos sin | T HQ HK D rot P |
#   q_st q_sh k_st k_sh v_st v_sh | page pages | kp_s0 kp_sh kp_ss vp_s0 vp_sh vp_ss | flags
pack_rotary = struct.Struct("@10P20qi0q").pack
# qik_page_pools: k v | layers pages heads page token_bytes | k layer, page, head bytes | v ...
pack_pools = struct.Struct("@2P11q").pack
# qik_paged_attn_args: q k_pages v_pages out page_table seq_lens query_starts | B T HQ HK D W
#   pages page max_new max_kv | q_st q_sh o_st o_sh table_st | kp_s0 kp_sh kp_ss vp_s0 vp_sh vp_ss |
#   sm_scale | window sinks flags
pack_paged_attn = struct.Struct("@7P21qf3i0q").pack
PAGED = 4    # QIK_ROTARY_PAGED
CAUSAL = 1   # QIK_PAGED_CAUSAL


@pytest.fixture
def cache(monkeypatch):
    """A cache on the CPU whose page copies are plain ones (the kernel needs a GPU)."""
    import qik.paged_kv as P

    def plain(k, v, moves):
        for p in (k, v):
            old = p.clone()
            for a, b, t in moves:
                p[:, b, :, :t] = old[:, a, :, :t]
    monkeypatch.setattr(P, "copy_pages", plain)

    def make(pages=12, page=16):
        c = P.PagedKVCache(1, pages, page, 1, 8, dtype=torch.float32, device="cpu")
        c.k_pages.zero_()  # (a new pool holds whatever the memory held, NaN too)
        c.v_pages.zero_()
        return c
    return make


def test_step_positions_slots_and_table(cache):
    c = cache()
    a, b = c.new_sequence(), c.new_sequence()
    s = c.step([a, b], [20, 3])
    assert s.seq_lens.tolist() == [20, 3] and s.query_starts.tolist() == [0, 20, 23]
    assert s.positions.tolist() == list(range(20)) + [0, 1, 2]
    assert s.page_table.tolist() == [[0, 1], [2, 0]]
    assert s.slots.tolist() == list(range(20)) + [32, 33, 34]
    assert (s.max_new, s.max_kv, s.tokens) == (20, 20, 23)
    s = c.step([b, a], [0, 1])
    assert s.slots.tolist() == [20] and s.positions.tolist() == [20] and s.query_starts.tolist() == [0, 0, 1]
    assert c.step([], []).seq_lens.shape == (0,)


def test_full_cache_changes_nothing(cache):
    from qik.paged_kv import CacheFull
    c = cache(pages=3)
    a, b = c.new_sequence(), c.new_sequence()
    c.step([a], [20])
    before = (c.free_pages, c.pages_of(a), c.length(a), c.length(b))
    with pytest.raises(CacheFull):
        c.step([a, b], [5, 17])
    with pytest.raises(CacheFull):
        c.fork(a, 2)
    assert before == (c.free_pages, c.pages_of(a), c.length(a), c.length(b)) and c.sequences() == [a, b]


def test_failed_copy_gives_its_pages_back(cache, monkeypatch):
    import qik.paged_kv as P
    c = cache()
    a = c.new_sequence()
    c.step([a], [20])
    monkeypatch.setattr(P, "copy_pages", lambda *x: (_ for _ in ()).throw(RuntimeError("no")))
    with pytest.raises(RuntimeError):
        c.fork(a)
    assert c.free_pages == 10 and c.sequences() == [a]


def test_fork_shares_full_pages_and_copies_the_rest(cache):
    c = cache()
    a = c.new_sequence()
    s = c.step([a], [40])
    c.k_pages[0, :, 0, :, 0] = torch.arange(12 * 16).view(12, 16).float()
    x, y = c.fork(a, 2)
    assert c.pages_of(x)[:2] == c.pages_of(a)[:2] and len({c.pages_of(i)[2] for i in (a, x, y)}) == 3
    assert torch.equal(c.k_pages[0, c.pages_of(x)[2], 0, :8], c.k_pages[0, s.page_table[0, 2], 0, :8])
    c.free(a)
    assert c.pages_of(x)[:2] == [0, 1] and c.free_pages == 12 - 4
    c.truncate(x, 20)  # page 1 is shared with y and no longer full: a copy
    assert c.pages_of(x)[0] == 0 and c.pages_of(x)[1] != 1 and c.pages_of(y)[1] == 1
    c.truncate(x, 16)
    assert c.pages_of(x) == [0]
    c.truncate(x, 0)
    assert c.pages_of(x) == [] and c.length(x) == 0
    full = c.new_sequence()
    c.step([full], [32])
    free = c.free_pages
    c.fork(full, 3)
    assert c.free_pages == free  # nothing partly filled, nothing copied


def test_compact_is_exact_under_random_use(cache):
    c, r = cache(pages=20), random.Random(1)
    from qik.paged_kv import CacheFull
    for _ in range(400):
        seqs = c.sequences()
        try:
            if not seqs or r.random() < 0.3:
                c.step([c.new_sequence()], [r.randint(1, 50)])
            elif r.random() < 0.4:
                c.fork(r.choice(seqs))
            elif r.random() < 0.5:
                c.truncate(s := r.choice(seqs), r.randint(0, c.length(s)))
            else:
                c.free(r.choice(seqs))
        except CacheFull:
            c.free(*c.sequences())
        before = {s: c.k_pages[:, c.pages_of(s)].clone() for s in c.sequences()}
        c.k_pages[:, [p for p in range(20) if c._users[p] == 0]] = -1
        c.compact()
        live = {p for s in c.sequences() for p in c.pages_of(s)}
        assert live == set(range(len(live))) and c.free_pages == 20 - len(live)
        users = [sum(p in c.pages_of(s) for s in c.sequences()) for p in range(20)]
        assert users == c._users
        for s, k in before.items():
            n = c.length(s)
            a, b = (t.transpose(1, 2).reshape(-1, 8)[:n] if n else None for t in (k[0], c.k_pages[0, c.pages_of(s)]))
            assert n == 0 or torch.equal(a, b)
        c.k_pages[:] = torch.rand(c.k_pages.shape)


def test_cache_refusals(cache):
    import qik.paged_kv as P
    for kw in (dict(page_size=24), dict(page_size=8), dict(num_pages=0)):
        with pytest.raises(ValueError):
            P.PagedKVCache(**(dict(num_layers=1, num_pages=2, page_size=16, num_kv_heads=1, head_dim=64, device="cpu") | kw))
    c = cache()
    a = c.new_sequence()
    for bad in (lambda: c.step([a, a], [1, 1]), lambda: c.step([a], [-1]), lambda: c.step([a], [1, 2]), lambda: c.truncate(a, 1),
                lambda: c.fork(a, -1), lambda: c.free(a, a)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: c.step([99], [1]), lambda: c.free(a, 99), lambda: c.fork(99), lambda: c.length(99)):
        with pytest.raises(KeyError):
            bad()
    assert c.sequences() == [a]


# ------------------------------------------------------------------------------ C entry points
@pytest.fixture(scope="module")
def lib():
    from qik import _lib as L
    return L.load(require_cuda=False)


def _fails(lib, rc, text):
    assert rc == 1 and text.encode() in lib.qik_last_error(), (rc, lib.qik_last_error())


def test_copy_pages_refuses_bad_moves(lib):
    """The list is checked before anything is launched."""
    p = pack_pools(4096, 8192, 2, 10, 2, 16, 128, 10 * 4096, 4096, 2048, 10 * 4096, 4096, 2048)

    def call(*moves, p=p):
        flat = (ctypes.c_int32 * (3 * len(moves)))(*[x for m in moves for x in m])
        return lib.qik_copy_pages(p, flat, len(moves), None)
    _fails(lib, call((0, 10, 1)), "outside 10 pages")
    _fails(lib, call((-1, 1, 1)), "outside 10 pages")
    _fails(lib, call((0, 1, 17)), "outside 10 pages")
    _fails(lib, call((0, 1, -1)), "outside 10 pages")
    _fails(lib, call((0, 2, 1), (1, 2, 1)), "page 2 is written twice")
    _fails(lib, call((0, 1, 1), (1, 2, 1)), "both read and written")
    _fails(lib, call((3, 3, 1)), "both read and written")
    assert call((0, 1, 0)) == 0  # nothing to copy
    assert lib.qik_copy_pages(p, None, 0, None) == 0
    _fails(lib, lib.qik_copy_pages(p, None, 1, None), "NULL")
    odd = pack_pools(4096, 8192, 2, 10, 2, 16, 100, 10 * 4096, 4096, 2048, 10 * 4096, 4096, 2048)
    _fails(lib, call((0, 1, 1), p=odd), "16 bytes")


def test_norm_entry_refusals(lib):
    x = ctypes.c_void_p(4096)

    def call(M=20, N=64, ldx=64, ldr=64, eps=1e-6, y=x, scale=x, ws=x):
        return lib.qik_add_rms_norm_e4m3(x, ldx, x, ldr, x, 0, M, N, eps, 0, x, y, scale, 0, ws, None)
    _fails(lib, call(N=60), "60 columns")
    _fails(lib, call(N=32776, ldx=32776), "32776 columns")
    _fails(lib, call(ldx=56), "pitches")
    _fails(lib, call(ldr=68), "pitches")
    _fails(lib, call(y=None), "NULL")
    _fails(lib, call(scale=None), "NULL")
    _fails(lib, call(ws=None), "NULL")
    _fails(lib, call(eps=-1.0), "eps")
    _fails(lib, call(y=ctypes.c_void_p(4104)), "aligned")
    assert call(M=0) == 0
    assert lib.qik_add_rms_norm_workspace_bytes(100, 64) >= 400 and lib.qik_add_rms_norm_workspace_bytes(3, 64) == 0


def test_rotary_entry_refusals(lib):
    def call(**kw):
        base = dict(q=4096, k=4096, v=4096, q_out=4096, k_out=4096, v_out=4096, positions=4096, slots=4096, cos=4096, sin=4096,
                    T=4, HQ=4, HK=2, D=128, rot=128, P=100, q_st=512, q_sh=128, k_st=256, k_sh=128, v_st=256, v_sh=128,
                    page=16, pages=4, kp_s0=4096, kp_sh=2048, kp_ss=128, vp_s0=4096, vp_sh=2048, vp_ss=128,
                    flags=PAGED)
        return lib.qik_rotary(pack_rotary(*[0 if x is None else x for x in (base | kw).values()]), None, None)
    for kw, text in ((dict(D=96), "head_dim"), (dict(rot=136), "rotated"), (dict(rot=24), "rotated"), (dict(P=0), "positions"),
                     (dict(q=None), "NULL"), (dict(v=None), "paged"), (dict(slots=None), "paged"), (dict(q_st=4), "strides"),
                     (dict(page=24), "power of two"), (dict(kp_ss=4), "page strides"), (dict(k=4100), "aligned"),
                     (dict(T=-1), "bad sizes")):
        _fails(lib, call(**kw), text)
    assert call(T=0) == 0


def test_attention_entry_refusals(lib):
    def call(ws=4096, ws_bytes=1 << 40, **kw):
        base = dict(q=4096, k_pages=4096, v_pages=4096, out=4096, page_table=4096, seq_lens=4096, query_starts=4096, B=2, T=4,
                    HQ=4, HK=2, D=128, W=10, pages=30, page=16, max_new=2, max_kv=160, q_st=512, q_sh=128, o_st=512, o_sh=128,
                    table_st=10, kp_s0=4096, kp_sh=2048, kp_ss=128, vp_s0=4096, vp_sh=2048, vp_ss=128, sm_scale=0.1,
                    window=0, sinks=0, flags=CAUSAL)
        a = pack_paged_attn(*[0 if x is None else x for x in (base | kw).values()])
        return lib.qik_paged_attention(a, ws, ws_bytes, None, None)
    for kw, text in ((dict(D=96), "head_dim"), (dict(HQ=5), "bad sizes"), (dict(page=24), "power of two"), (dict(page=8), "power of two"),
                     (dict(W=1 << 27), "page table"), (dict(max_new=5), "max_new"), (dict(max_kv=-1), "max_kv"),
                     (dict(window=-1), "window"), (dict(window=4, flags=0), "causal"), (dict(sm_scale=0.0), "sm_scale"),
                     (dict(sm_scale=float("nan")), "sm_scale"), (dict(q=None), "NULL"), (dict(page_table=None), "NULL"),
                     (dict(out=4104), "aligned"), (dict(q_sh=4), "strides"), (dict(max_kv=100000, ws_bytes=10), "workspace"),
                     (dict(max_kv=100000, ws=None), "workspace"), (dict(B=-1), "bad sizes")):
        _fails(lib, call(**kw), text)
    assert call(T=0, max_new=0) == 0 and call(B=0) == 0


def test_calls_need_a_gpu():
    from qik.paged_attention import paged_attention
    from qik.paged_kv import copy_pages
    from qik.rms_norm import fused_add_rms_norm, fused_add_rms_norm_e4m3
    from qik.rotary import apply_rotary
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: fused_add_rms_norm(x, x, x[0], 1e-6), lambda: fused_add_rms_norm_e4m3(x, x, x[0], 1e-6),
                 lambda: apply_rotary(x[:, None], x[:, None], i, (x.float(), x.float())),
                 lambda: copy_pages(x[None, None, None], x[None, None, None], [(0, 0, 0)]),
                 lambda: paged_attention(x[:, None], x[None, None], x[None, None], i[:, None], i, i, 1)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------ rotary tables
def test_rotary_scalings():
    from qik.rotary import rotary_frequencies, rotary_table
    f, gain = rotary_frequencies(64, base=1e4)
    assert gain == 1 and f.dtype == torch.float64 and f[0] == 1 and math.isclose(f[-1], 1e4 ** (-62 / 64))
    lin, _ = rotary_frequencies(64, base=1e4, scaling="linear", factor=8.0)
    assert torch.equal(lin, f / 8)
    ntk, _ = rotary_frequencies(64, base=1e4, scaling="ntk", factor=8.0)
    assert ntk[0] == 1 and math.isclose(ntk[-1], f[-1] / 8, rel_tol=1e-12)
    for name in ("yarn", "bands"):
        g, gain = rotary_frequencies(64, base=1e4, scaling=name, factor=8.0, original_positions=4096)
        assert math.isclose(g[0], f[0]) and math.isclose(g[-1], f[-1] / 8) and ((g <= f) & (g >= f / 8 * (1 - 1e-12))).all()
        assert (g[1:] < g[:-1]).all() and math.isclose(gain, 0.1 * math.log(8) + 1 if name == "yarn" else 1)
    cos, sin = rotary_table(32, 200, device="cpu", base=100.0)
    p, i = 171, 5
    assert cos.shape == (200, 16) and math.isclose(cos[p, i], math.cos(p * 100.0 ** (-2 * i / 32)), abs_tol=1e-7)
    assert math.isclose(sin[p, i], math.sin(p * 100.0 ** (-2 * i / 32)), abs_tol=1e-7)
    for kw in (dict(scaling="other"), dict(factor=0.0), dict(base=1.0), dict(original_positions=0)):
        with pytest.raises(ValueError):
            rotary_frequencies(64, **kw)
    with pytest.raises(ValueError):
        rotary_frequencies(63)
    with pytest.raises(ValueError):
        rotary_table(64, 0, device="cpu")


def test_packed_structs_match_the_header(tmp_path):
    """The packers above lay their fields out as a C compiler lays out include/qik.h."""
    import subprocess

    from conftest import ROOT
    c = tmp_path / "sizes.c"
    c.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "qik.h"\nint main(void) {\n'
                 'printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(qik_rotary_args), offsetof(qik_rotary_args, kp_s0), '
                 'sizeof(qik_page_pools), sizeof(qik_paged_attn_args), offsetof(qik_paged_attn_args, sm_scale), '
                 'offsetof(qik_paged_attn_args, max_kv));\nreturn 0;\n}\n')
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(c), "-o", str(tmp_path / "sizes")], check=True)
    said = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()]
    rotary = pack_rotary(*range(1, 32))
    attn = pack_paged_attn(*range(1, 29), 0.5, *range(30, 33))
    assert said[0] == len(rotary) and int.from_bytes(rotary[said[1]:said[1] + 8], "little") == 25
    assert said[2] == len(pack_pools(*range(13))) and said[3] == len(attn)
    assert struct.unpack_from("f", attn, said[4])[0] == 0.5 and int.from_bytes(attn[said[5]:said[5] + 8], "little") == 17
