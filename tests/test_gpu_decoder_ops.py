"""GPU: residual + RMS norm, rotary positions and page copies against the definitions in 64 bits.

Bounds: one rounding to the output's type is half a step (eps / 2 of the value; e4m3: 2^-4, or
2^-10 below its normal range); the fp32 work in between stays under 1e-5 relative (a sum of N
squares in per-thread chains of at most 32 and trees: (32 + 10) * 2^-24 < 3e-6).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def norm_exact(x, r, w, eps):
    h = x.double() + (0 if r is None else r.double())
    return h, h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()


def close(got, want, half, rel=1e-5, tiny=0.0):
    off = (got.double() - want).abs()
    assert (off <= (half + rel) * want.abs() + tiny).all(), (off - (half + rel) * want.abs()).max().item()


NORMS = [(1, 8), (1, 4096), (3, 64), (2, 512), (5, 520), (77, 1536), (300, 5120), (2500, 1000), (9, 16384), (4, 16392),
         (3, 32768), (40, 24)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N", NORMS)
def test_add_rms_norm(M, N, dtype):
    from qik.rms_norm import fused_add_rms_norm, fused_add_rms_norm_e4m3
    g = gen(M + N)
    x = torch.randn(M, N, generator=g, device=DEV).to(dtype)
    r = (torch.randn(M, N, generator=g, device=DEV) * 5).to(dtype)
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for weight in (torch.randn(N, generator=g, device=DEV).to(dtype), torch.randn(N, generator=g, device=DEV)):
        for res in (r, None):
            h, y = norm_exact(x, res, weight, 1e-6)
            got, s = fused_add_rms_norm(x, res, weight, 1e-6)
            close(got, y, half, tiny=tiny)
            if res is None:
                assert s is x
            else:
                close(s, h, half, rel=0, tiny=tiny)
            for scales in ("tensor", "row"):
                q, scale, s2 = fused_add_rms_norm_e4m3(x, res, weight, 1e-6, scales=scales)
                assert torch.equal(s2, s) and q.dtype == torch.float8_e4m3fn
                top = y.abs().amax(-1) if scales == "row" else y.abs().amax().reshape(1)
                close(scale, (top / 448).clamp_min(1e-12), 0)
                step = scale.double()[:, None] if scales == "row" else scale.double()
                close(q.float(), y / step, 2.0 ** -4, rel=2e-5, tiny=2.0 ** -10)
                assert q.float().abs().max() == 448


def test_norm_codes_feed_the_fp8_linear():
    """The whole-tensor codes and scale are what FP8Linear.forward_e4m3 takes."""
    from qik.fp8 import FP8Linear, quantize_weight_tensorwise
    from qik.rms_norm import fused_add_rms_norm_e4m3
    g = gen(5)
    x, r = (torch.randn(50, 512, generator=g, device=DEV).bfloat16() for _ in range(2))
    w = torch.randn(512, generator=g, device=DEV).bfloat16()
    lin = FP8Linear(512, 256).to(DEV)
    wq, sw = quantize_weight_tensorwise((torch.randn(256, 512, generator=g, device=DEV) * 0.05).bfloat16())
    lin.weight.copy_(wq)
    lin.weight_scale.copy_(sw)
    q, s, _ = fused_add_rms_norm_e4m3(x, r, w, 1e-6)
    got = lin.forward_e4m3(q, s).double()
    want = (q.double() * s.double()) @ (wq.double() * sw.double()).T
    assert ((got - want).norm() / want.norm()).item() < 5e-3


@pytest.mark.parametrize("scales", ["tensor", "row"])
def test_norm_extremes(scales):
    """Rows of zeros, infinities and NaN: the scale floor, and NaN where the plain form has it."""
    from qik.rms_norm import fused_add_rms_norm, fused_add_rms_norm_e4m3
    z = torch.zeros(3, 64, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    q, s, h = fused_add_rms_norm_e4m3(z, z, w, 1e-6, scales=scales)
    assert (q.float() == 0).all() and torch.allclose(s, torch.full_like(s, 1e-12)) and (h == 0).all()
    x = torch.randn(3, 64, device=DEV).bfloat16()
    x[1, 5] = float("nan")
    y, _ = fused_add_rms_norm(x, None, w, 1e-6)
    assert y[1].isnan().all() and y[0].isfinite().all() and y[2].isfinite().all()
    q, s, _ = fused_add_rms_norm_e4m3(x, None, w, 1e-6, scales=scales)
    if scales == "row":
        assert s[1].isnan() and s[0].isfinite() and q[0].float().isfinite().all() and q[1].float().isnan().all()
    else:
        assert s.isnan().all() and q.float().isnan().all()
    x[1, 5] = float("inf")  # 1 / rms is 0 and inf * 0 NaN, as the plain form has it
    y, _ = fused_add_rms_norm(x, None, w, 1e-6)
    assert y[1, 5].isnan() and (y[1, :5] == 0).all()


def test_norm_strides_shapes_and_streams():
    from qik.rms_norm import fused_add_rms_norm, fused_add_rms_norm_e4m3
    g = gen(6)
    wide = torch.randn(40, 256, generator=g, device=DEV).bfloat16()
    w = torch.randn(128, generator=g, device=DEV).bfloat16()
    for x in (wide[:, 8:136], wide[:, 3:131], wide.view(5, 8, 256)[..., :128], wide[::3, :128]):
        r = torch.randn(x.shape, generator=g, device=DEV).bfloat16()
        h, y = norm_exact(x, r, w, 1e-5)
        a, s = fused_add_rms_norm(x, r, w, 1e-5)
        assert a.shape == x.shape
        close(a, y, 2.0 ** -8)
        close(s, h, 2.0 ** -8, rel=0)
    x = torch.randn(64, 128, generator=g, device=DEV).bfloat16()
    want = fused_add_rms_norm_e4m3(x, x, w, 1e-6)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append(fused_add_rms_norm_e4m3(x, x, w, 1e-6))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got.append(fused_add_rms_norm_e4m3(x, x, w, 1e-6))
    graph.replay()
    torch.cuda.synchronize()
    for q, s, h in got:
        assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s, want[1]) and torch.equal(h, want[2])
    q, s, h = fused_add_rms_norm_e4m3(x[:0], x[:0], w, 1e-6)
    assert q.shape == (0, 128) and s.shape == (1,)


# ------------------------------------------------------------------------------ rotary
def turn_exact(x, pos, rot, interleaved, f, gain):
    x = x.double()
    ang = pos.double()[:, None, None] * f.to(DEV)
    c, s = gain * ang.cos(), gain * ang.sin()
    y = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,HK,D,rot", [(1, 1, 1, 64, 64), (5, 4, 2, 128, 128), (33, 32, 8, 128, 96), (200, 7, 1, 64, 16),
                                          (1001, 3, 3, 128, 64), (17, 2, 1, 256, 256), (9, 5, 5, 256, 48)])
def test_rotary(T, H, HK, D, rot, interleaved, dtype):
    from qik.rotary import apply_rotary, rotary_frequencies, rotary_store, rotary_table
    g = gen(T + D)
    kw = dict(base=1e6, scaling=("none", "linear", "ntk", "yarn", "bands")[T % 5], factor=4.0, original_positions=2048)
    far = 100000
    table = rotary_table(rot, far, **kw)
    f, gain = rotary_frequencies(rot, **kw)
    qkv = torch.randn(T, (H + 2 * HK) * D, generator=g, device=DEV).to(dtype)
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([H * D, HK * D, HK * D], 1))
    half = torch.finfo(dtype).eps / 2
    tiny = 1e-6 + (2.0 ** -25 if dtype == torch.float16 else 0)  # |x| < 6: 2^-22 of the products
    for kind in (torch.int32, torch.int64):
        pos = torch.randint(0, far, (T,), generator=g, device=DEV).to(kind)
        qt, kt = apply_rotary(q, k, pos, table, interleaved=interleaved)
        want_q, want_k = (turn_exact(t, pos, rot, interleaved, f, gain) for t in (q, k))
        close(qt, want_q, half, rel=0, tiny=4 * tiny)
        close(kt, want_k, half, rel=0, tiny=4 * tiny)
        page = (16, 32, 64)[T % 3]
        pages = T // page + 4
        kp, vp = (torch.randn(pages, HK, page, D, generator=g, device=DEV).to(dtype) for _ in range(2))
        kp0, vp0 = kp.clone(), vp.clone()
        slots = torch.randperm(pages * page, generator=g, device=DEV)[:T].to(kind)
        if T > 4:
            slots[3] = -1  # padding
        q2 = rotary_store(q, k, v, pos, table, slots, kp, vp, interleaved=interleaved)
        assert torch.equal(q2, qt)
        keep = slots >= 0
        kp0[(slots[keep] // page).long(), :, (slots[keep] % page).long()] = kt[keep]
        vp0[(slots[keep] // page).long(), :, (slots[keep] % page).long()] = v[keep]
        assert torch.equal(kp, kp0) and torch.equal(vp, vp0)


def test_rotary_bad_indices_are_skipped_and_reported():
    from qik import _lib as L
    from qik.rotary import apply_rotary, rotary_store, rotary_table
    dev = torch.device(DEV, 0)
    table = rotary_table(64, 50)
    q = torch.randn(4, 2, 64, device=DEV).bfloat16()
    k = torch.randn(4, 1, 64, device=DEV).bfloat16()
    pos = torch.tensor([0, 50, -1, 49], device=DEV)
    qt, kt = apply_rotary(q, k, pos, table)
    torch.cuda.synchronize()
    assert L.device_status(dev) == L.STATUS_BAD_INDEX
    L.status_word(dev).zero_()
    assert (qt[1:3] == 0).all() and (kt[1:3] == 0).all() and (qt[3] != 0).any() and torch.equal(qt[0], q[0])
    kp, vp = torch.zeros(2, 1, 16, 64, device=DEV).bfloat16(), torch.zeros(2, 1, 16, 64, device=DEV).bfloat16()
    rotary_store(q, k, k, torch.zeros(4, dtype=torch.int32, device=DEV), table, torch.tensor([32, -7, 5, 10 ** 12], device=DEV), kp, vp)
    torch.cuda.synchronize()
    assert L.device_status(dev) == L.STATUS_BAD_INDEX
    L.status_word(dev).zero_()
    assert torch.equal(kp[0, :, 5], k[2]) and (kp != 0).sum() == (k[2] != 0).sum() and (vp != 0).sum() == (k[2] != 0).sum()
    assert apply_rotary(q[:0], k[:0], pos[:0], table)[0].shape == (0, 2, 64)


# ------------------------------------------------------------------------------ pages
@pytest.mark.parametrize("L_,N,H,page,D,n", [(1, 4, 1, 16, 64, 1), (3, 40, 2, 32, 128, 19), (2, 900, 1, 16, 64, 400), (2, 30, 8, 128, 128, 9)])
def test_copy_pages(L_, N, H, page, D, n):
    import random
    from qik.paged_kv import copy_pages
    g, r = gen(N), random.Random(N)
    k, v = (torch.randn(L_, N, H, page, D, generator=g, device=DEV).bfloat16() for _ in range(2))
    ids = r.sample(range(N), n + max(1, n // 2))
    moves = [(ids[n + r.randrange(max(1, n // 2))], ids[i], r.choice((0, 1, page // 2 + 1, page))) for i in range(n)]
    want = [k.clone(), v.clone()]
    for p, w in zip((k, v), want):
        for a, b, t in moves:
            w[:, b, :, :t] = p[:, a, :, :t]
    copy_pages(k, v, moves)
    torch.cuda.synchronize()
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    one = k[0].clone()
    copy_pages(k[0], v[0], moves[:1])  # one layer's pools
    one[moves[0][1], :, :moves[0][2]] = one[moves[0][0], :, :moves[0][2]]
    assert torch.equal(k[0], one)


def test_sequences_keep_their_tokens():
    """fork, truncate, free and compact against a plain list of tokens per sequence."""
    import random
    from qik.paged_kv import CacheFull, PagedKVCache
    r = random.Random(3)
    c = PagedKVCache(2, 40, 16, 2, 64, device=DEV)
    c.k_pages.zero_(), c.v_pages.zero_()
    told, stamp = {}, 0
    for _ in range(300):
        op = r.random()
        seqs = c.sequences()
        try:
            if op < 0.2 or not seqs:
                told[c.new_sequence()] = []
            elif op < 0.6:
                some = r.sample(seqs, r.randint(1, min(3, len(seqs))))
                counts = [r.randint(0, 20) for _ in some]
                step = c.step(some, counts)
                n = sum(counts)
                vals = torch.arange(stamp, stamp + n, device=DEV, dtype=torch.float32) % 251
                stamp += n
                page, at = step.slots // 16, step.slots % 16
                c.k_pages[:, page, :, at] = vals.bfloat16()[:, None, None, None].expand(n, 2, 2, 64)
                c.v_pages[:, page, :, at] = -vals.bfloat16()[:, None, None, None].expand(n, 2, 2, 64)
                for s, m, part in zip(some, counts, vals.split(counts)):
                    told[s] = told[s] + part.tolist()
                assert step.positions.tolist() == [p for s, m in zip(some, counts) for p in range(len(told[s]) - m, len(told[s]))]
            elif op < 0.75:
                s = r.choice(seqs)
                for child in c.fork(s, r.randint(0, 2)):
                    told[child] = list(told[s])
            elif op < 0.85:
                s = r.choice(seqs)
                m = r.randint(0, c.length(s))
                c.truncate(s, m)
                told[s] = told[s][:m]
            elif op < 0.95:
                s = r.choice(seqs)
                c.free(s)
                del told[s]
            else:
                c.compact()
                live = c.num_pages - c.free_pages
                assert all(p < live for s in c.sequences() for p in c.pages_of(s))
        except CacheFull:
            s = r.choice(seqs)
            c.free(s)
            del told[s]
        for s in c.sequences():
            assert c.length(s) == len(told[s])
            pages = c.pages_of(s)
            got = torch.cat([c.k_pages[:, p].transpose(1, 2) for p in pages], 1)[:, :len(told[s])] if pages else c.k_pages[:, 0, 0, :0, None]
            want = torch.tensor(told[s], device=DEV).bfloat16()[None, :, None, None]
            assert (got == want).all()
    c.free(*c.sequences())
    assert c.free_pages == 40


def test_a_decoder_step_over_the_paged_cache():
    """Norm -> FP8 QKV -> rotary + store -> attention -> FP8 out, prompt then single tokens then a
    fork, against the same step composed in 64 bits from this step's own intermediates."""
    from qik.fp8 import FP8Linear, quantize_weight_tensorwise
    from qik.paged_attention import paged_attention
    from qik.paged_kv import PagedKVCache
    from qik.rms_norm import fused_add_rms_norm_e4m3
    from qik.rotary import rotary_frequencies, rotary_store, rotary_table
    from test_gpu_paged_attention import check, exact
    g = gen(40)
    C, H, HK, D = 512, 8, 2, 64
    qkv_lin, out_lin = FP8Linear(C, (H + 2 * HK) * D).to(DEV), FP8Linear(H * D, C).to(DEV)
    for lin in (qkv_lin, out_lin):
        w, s = quantize_weight_tensorwise((torch.randn(lin.weight.shape, generator=g, device=DEV) * 0.05).bfloat16())
        lin.weight.copy_(w)
        lin.weight_scale.copy_(s)
    weight = torch.ones(C, device=DEV).bfloat16()
    cache = PagedKVCache(1, 64, 16, HK, D, device=DEV)
    table = rotary_table(D, 4096, base=1e5)
    f, gain = rotary_frequencies(D, base=1e5)
    kp, vp = cache.layer(0)
    a, b = cache.new_sequence(), cache.new_sequence()

    def forward(seqs, counts):
        step = cache.step(seqs, counts)
        x, res = (torch.randn(step.tokens, C, generator=g, device=DEV).bfloat16() for _ in range(2))
        codes, scale, res = fused_add_rms_norm_e4m3(x, res, weight, 1e-6)
        qkv = qkv_lin.forward_e4m3(codes, scale)
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([H * D, HK * D, HK * D], 1))
        qt = rotary_store(q, k, v, step.positions, table, step.slots, kp, vp)
        o = paged_attention(qt, kp, vp, step.page_table, step.seq_lens, step.query_starts, step.max_new, max_kv=step.max_kv)
        y = out_lin(o.flatten(1))
        want_q = turn_exact(q, step.positions, D, False, f, gain)
        close(qt, want_q, 2.0 ** -8, rel=0, tiny=1e-5)
        close(kp[step.slots // 16, :, step.slots % 16], turn_exact(k, step.positions, D, False, f, gain), 2.0 ** -8, rel=0, tiny=1e-5)
        assert torch.equal(vp[step.slots // 16, :, step.slots % 16], v)
        s = dict(q=qt, k_pages=kp, v_pages=vp, page_table=step.page_table)
        check(o, s, counts, [cache.length(i) for i in seqs])
        assert y.shape == (step.tokens, C) and y.isfinite().all()
        return o

    forward([a, b], [37, 5])
    forward([a, b], [1, 1])
    (c,) = cache.fork(a)
    cache.free(b)
    cache.compact()
    forward([c, a], [1, 3])
    forward([a, c], [90, 1])
