"""GPU: paged attention within the bound that its arithmetic gives, element by element, in fp16 and bf16.

With half = eps / 2 of the type and, per output element, mass = sum p |v| / sum p:
* p is rounded to the type before p . v: half of each term; in fp16 a p below 2^-14 by up to 2^-25
  absolute, in units in which the kernel's sum of p is at least sum p / max p: 2^-25 sum |v| / (sum p / max p);
* a score's error moves its p, in the product and in the sum: twice (D / 16 + 2) 2^-22 sum |q k| scale for
  the tensor core's fp32 additions of 16 products each and the joining of two chains, 2^-21 for 2^x and
  2^-23 (|score - max| log2(e) + 1) for the exponent's rounding, which stays under 2^-18 where p is above 2^-25;
* both sums are chains of at most kv / 16 + 64 fp32 additions (a lane has 4 of a tile's 64 keys, a matrix
  instruction 16; joins of warps and pieces): 2^-23 each, for the product and for the sum;
* the result is rounded once: half of it, 2^-25 at least in fp16.
"""
import math

import pytest
import torch

from test_gpu_paged_attention import DEV, make, run

pytestmark = pytest.mark.gpu


def bounded(got, s, new, kv, causal=True):
    D, H, HK, page = s["q"].shape[2], s["q"].shape[1], s["k_pages"].shape[1], s["k_pages"].shape[2]
    scale, half = D ** -0.5, torch.finfo(got.dtype).eps / 2
    table, at, worst = s["page_table"].cpu().long(), 0, 0.0
    for i, (n, m) in enumerate(zip(new, kv)):
        t = torch.arange(m)
        where = (table[i][t // page].to(DEV), (t % page).to(DEV))
        k, v = (p[where[0], :, where[1]].double().repeat_interleave(H // HK, 1) for p in (s["k_pages"], s["v_pages"]))
        q = s["q"][at:at + n].double()
        t = t.to(DEV)
        last = m - n + torch.arange(n, device=DEV) if causal else torch.full((n,), m - 1, device=DEV)
        seen = t[None] <= last[:, None]
        a = (torch.einsum("nhd,mhd->hnm", q, k) * scale).masked_fill(~seen, -math.inf)
        size = torch.einsum("nhd,mhd->hnm", q.abs(), k.abs()) * scale
        p = torch.exp(a - a.amax(-1, keepdim=True))
        total = p.sum(-1)[..., None]
        p = p / total
        moved = p * (2 * (D / 16 + 2) * 2.0 ** -22 * size + 2.0 ** -18)
        want, mass, move = (torch.einsum("hnm,mhd->nhd", x, y) for x, y in ((p, v), (p, v.abs()), (moved, v.abs())))
        move = move + moved.sum(-1).T[..., None] * want.abs()  # in the product, and in the sum
        chain = 2 * (m / 16 + 64) * 2.0 ** -23
        tiny = 2.0 ** -25 * torch.einsum("nm,mhd->nhd", seen.double(), v.abs()) / total[..., 0].T[..., None] + 2.0 ** -25 if got.dtype == torch.float16 else 0.0
        bound = (half + chain) * mass + move + half * want.abs() + tiny
        worst = max(worst, ((got[at:at + n].double() - want).abs() / bound).max().item())
        at += n
    assert worst <= 1.0, f"{worst} of the bound"


CALLS = [([1], [300], 32, 8), ([1, 1, 1], [17, 900, 4000], 8, 8), ([3, 1, 16], [3, 700, 1000], 4, 1), ([13], [2000], 5, 1), ([1], [30000], 8, 1),
         ([100], [1000], 8, 2), ([257, 64, 300], [257, 640, 1300], 3, 1), ([130, 33], [4130, 2033], 28, 4), ([700], [700], 5, 5), ([513], [9000], 4, 4)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("call", range(len(CALLS)))
def test_within_the_bound(call, dim, dtype):
    new, kv, H, HK = CALLS[call]
    s = make(new, kv, H, HK, dim, (64, 16, 128, 32, 256)[call % 5], dtype, seed=110 + call)
    bounded(run(s), s, new, kv)
    bounded(run(s, causal=False), s, new, kv, causal=False)
