// qik_rotary.cu -- rotary positions of q and k, with the rotated k and v stored into the
// pages of a cache.
//
//   pair (a, b) of a head -> (a cos - b sin, b cos + a sin), cos and sin from row
//   positions[t] of two fp32 tables [P, rot / 2]; pairs are (2i, 2i + 1) (interleaved)
//   or (i, i + rot / 2) (halves) of the head's first `rot` columns, the rest of the
//   head is copied.  fp32 arithmetic, one rounding to the tensors' type.
//
// The table is filled once by the caller from angles in 64 bits: at far positions an
// fp32 angle has lost the digits that a cosine needs, and the kernel then computes no
// trigonometry.  Bound by HBM: each of q, k and v is read and written once; the table
// rows are a few percent of that and stay in L2.  One warp takes 16 heads of one token
// in four steps whose loads are all in flight before the first is used: one task shape
// for a decode step (many small independent tasks) and a prompt alike.  A lane holds 8
// pairs of a head (two 16-byte vectors), so its 8 cosines and sines serve its 4 heads.
#include "qik_device.cuh"
#include "qik_host.h"

namespace qik {

constexpr int kRotaryWarps = 4;
constexpr int kRotarySteps = 4;

struct RotaryDev {
  const uint16_t *q, *k, *v;
  uint16_t *q_out, *k_out, *v_out;
  const void *positions, *slots;
  const float *cos, *sin;
  int* status;
  int64_t T, q_st, k_st, v_st;       // token strides (elements)
  int64_t q_sh, k_sh, v_sh;          // head strides
  int64_t kp_s0, kp_sh, kp_ss;       // k pages: page, head, token strides
  int64_t vp_s0, vp_sh, vp_ss;
  int64_t n_slots;
  int P, HQ, HK, HV, D, rot, page_log2, tasks_per_token;
  bool interleaved, pos64, slot64, paged;
};

template <bool F16>
__device__ __forceinline__ void rot_unpack(uint32_t w, float& a, float& b) {
  if (F16) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = p.x;
    b = p.y;
  } else {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xFFFF0000u);
  }
}
template <bool F16>
__device__ __forceinline__ uint32_t rot_pack(float a, float b) {
  return F16 ? pack_f16x2(a, b) : pack_bf16x2(a, b);
}
__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, bool wide) {
  return wide ? __ldg(static_cast<const long long*>(p) + i) : static_cast<int64_t>(__ldg(static_cast<const int*>(p) + i));
}

// ITEMS = D / 16 lanes a head, two 16-byte vectors each, laid so that neighbouring lanes read
// neighbouring vectors.  Streaming loads and stores: 8111 tokens of 72 heads (301 MB) take 49.9 us
// (6.04 TB/s), 55.0 without the hints.
// Halves: lane item i < rot / 16 holds columns 8i .. 8i + 7 and their partners rot / 2 on, the
// others the copied columns.  Interleaved: columns 8i .. and D / 2 + 8i .., either turned or not.
template <bool F16, int ITEMS>
__global__ void __launch_bounds__(kRotaryWarps * 32) rotary_kernel(const RotaryDev a) {
  constexpr int kHeadsPerStep = 32 / ITEMS;
  const int lane = threadIdx.x & 31;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * kRotaryWarps + (threadIdx.x >> 5);
  const int64_t t = task / a.tasks_per_token;
  pdl_wait();
  if (t >= a.T) return;
  const int item = lane % ITEMS;
  const int head0 = static_cast<int>(task % a.tasks_per_token) * (kHeadsPerStep * kRotarySteps) + lane / ITEMS;
  const int heads = a.HQ + a.HK + a.HV;
  const int half = a.rot / 2;
  const int turned_items = a.rot / 16;
  int c0 = 8 * item, c1;  // first columns of the two vectors
  bool t0, t1;            // turned
  if (a.interleaved) {
    c1 = a.D / 2 + c0;
    t0 = c0 < a.rot;
    t1 = c1 < a.rot;
  } else {
    t0 = t1 = item < turned_items;
    c1 = c0 + half;
    if (!t0) {
      c0 = a.rot + 8 * (item - turned_items);
      c1 = c0 + (a.D - a.rot) / 2;
    }
  }

  const int64_t pos = load_index(a.positions, t, a.pos64);
  const bool pos_ok = pos >= 0 && pos < a.P;
  int64_t slot = -1;
  bool store = !a.paged;
  if (a.paged) {
    slot = load_index(a.slots, t, a.slot64);
    store = slot >= 0 && slot < a.n_slots && pos_ok;
    if (slot >= a.n_slots && lane == 0) report_bad_index(a.status);
  }
  if (!pos_ok && lane == 0) report_bad_index(a.status);
  const int64_t pg = store && a.paged ? slot >> a.page_log2 : 0;
  const int64_t in_page = store && a.paged ? slot & ((1 << a.page_log2) - 1) : t;

  uint4 v0[kRotarySteps], v1[kRotarySteps];
#pragma unroll
  for (int s = 0; s < kRotarySteps; ++s) {
    const int hd = head0 + s * kHeadsPerStep;
    if (hd < heads) {
      const uint16_t* src = hd < a.HQ            ? a.q + t * a.q_st + hd * a.q_sh
                            : hd < a.HQ + a.HK ? a.k + t * a.k_st + (hd - a.HQ) * a.k_sh
                                                 : a.v + t * a.v_st + (hd - a.HQ - a.HK) * a.v_sh;
      v0[s] = __ldcs(reinterpret_cast<const uint4*>(src + c0));
      v1[s] = __ldcs(reinterpret_cast<const uint4*>(src + c1));
    }
  }
  // eight angles: those of the 8 pairs (halves), or of the 4 pairs of each vector
  float c[8], sn[8];
  {
    const int p0 = a.interleaved ? c0 / 2 : c0, p1 = a.interleaved ? c1 / 2 : c0 + 4;
    float4 ca = make_float4(1.0f, 1.0f, 1.0f, 1.0f), sa = make_float4(0.0f, 0.0f, 0.0f, 0.0f), cb = ca, sb = sa;
    if (t0 && pos_ok) {
      ca = __ldg(reinterpret_cast<const float4*>(a.cos + pos * half + p0));
      sa = __ldg(reinterpret_cast<const float4*>(a.sin + pos * half + p0));
    }
    if (t1 && pos_ok) {
      cb = __ldg(reinterpret_cast<const float4*>(a.cos + pos * half + p1));
      sb = __ldg(reinterpret_cast<const float4*>(a.sin + pos * half + p1));
    }
    c[0] = ca.x, c[1] = ca.y, c[2] = ca.z, c[3] = ca.w, c[4] = cb.x, c[5] = cb.y, c[6] = cb.z, c[7] = cb.w;
    sn[0] = sa.x, sn[1] = sa.y, sn[2] = sa.z, sn[3] = sa.w, sn[4] = sb.x, sn[5] = sb.y, sn[6] = sb.z, sn[7] = sb.w;
  }
#pragma unroll
  for (int s = 0; s < kRotarySteps; ++s) {
    const int hd = head0 + s * kHeadsPerStep;
    if (hd >= heads) continue;
    const bool is_q = hd < a.HQ, is_k = !is_q && hd < a.HQ + a.HK;
    uint32_t w0[4] = {v0[s].x, v0[s].y, v0[s].z, v0[s].w}, w1[4] = {v1[s].x, v1[s].y, v1[s].z, v1[s].w};
    if (is_q || is_k) {
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x, y;
          if (t0) {
            rot_unpack<F16>(w0[i], x, y);
            w0[i] = rot_pack<F16>(fmaf(x, c[i], -(y * sn[i])), fmaf(y, c[i], x * sn[i]));
          }
          if (t1) {
            rot_unpack<F16>(w1[i], x, y);
            w1[i] = rot_pack<F16>(fmaf(x, c[4 + i], -(y * sn[4 + i])), fmaf(y, c[4 + i], x * sn[4 + i]));
          }
        }
      } else if (t0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x0, x1, y0, y1;
          rot_unpack<F16>(w0[i], x0, x1);
          rot_unpack<F16>(w1[i], y0, y1);
          w0[i] = rot_pack<F16>(fmaf(x0, c[2 * i], -(y0 * sn[2 * i])), fmaf(x1, c[2 * i + 1], -(y1 * sn[2 * i + 1])));
          w1[i] = rot_pack<F16>(fmaf(y0, c[2 * i], x0 * sn[2 * i]), fmaf(y1, c[2 * i + 1], x1 * sn[2 * i + 1]));
        }
      }
    }
    if (!pos_ok) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w0[i] = w1[i] = 0u;
    }
    uint16_t* dst;
    if (is_q) {
      dst = a.q_out + (t * a.HQ + hd) * a.D;
    } else if (!store) {
      continue;
    } else if (is_k) {
      dst = a.k_out + pg * a.kp_s0 + (hd - a.HQ) * a.kp_sh + in_page * a.kp_ss;
    } else {
      dst = a.v_out + pg * a.vp_s0 + (hd - a.HQ - a.HK) * a.vp_sh + in_page * a.vp_ss;
    }
    __stcs(reinterpret_cast<uint4*>(dst + c0), make_uint4(w0[0], w0[1], w0[2], w0[3]));
    __stcs(reinterpret_cast<uint4*>(dst + c1), make_uint4(w1[0], w1[1], w1[2], w1[3]));
  }
  pdl_trigger();
}

}  // namespace qik

using namespace qik;

extern "C" int qik_rotary(const qik_rotary_args* args, int* status, void* stream) {
  QIK_REQUIRE(args != nullptr, "qik_rotary: args is NULL");
  const qik_rotary_args& A = *args;
  QIK_REQUIRE(A.T >= 0 && A.T <= 0x7FFFFFFFll && A.HQ >= 0 && A.HK >= 0 && A.HQ + A.HK > 0 && A.HQ <= 4096 && A.HK <= 4096,
              "qik_rotary: bad sizes (T=%lld, %lld + %lld heads)", (long long)A.T, (long long)A.HQ, (long long)A.HK);
  QIK_REQUIRE(A.D == 64 || A.D == 128 || A.D == 256, "qik_rotary: head_dim %lld unsupported (64, 128 or 256)",
              (long long)A.D);
  QIK_REQUIRE(A.rot > 0 && A.rot <= A.D && A.rot % 16 == 0, "qik_rotary: %lld rotated columns of %lld (a multiple of 16)",
              (long long)A.rot, (long long)A.D);
  QIK_REQUIRE(A.P > 0 && A.P <= (1ll << 30), "qik_rotary: table of %lld positions", (long long)A.P);
  const bool paged = (A.flags & QIK_ROTARY_PAGED) != 0;
  if (A.T == 0) return QIK_OK;
  QIK_REQUIRE((A.HQ == 0 || (A.q && A.q_out)) && (A.HK == 0 || (A.k && A.k_out)) && A.positions && A.cos && A.sin,
              "qik_rotary: NULL pointer");
  QIK_REQUIRE(!paged || (A.HK > 0 && A.v && A.v_out && A.slots), "qik_rotary: the paged form needs k, v, pages and slots");
  QIK_REQUIRE(aligned16(A.q) && aligned16(A.k) && aligned16(A.v) && aligned16(A.q_out) && aligned16(A.k_out) &&
                  aligned16(A.v_out) && aligned16(A.cos) && aligned16(A.sin),
              "qik_rotary: pointers must be 16-byte aligned");
  QIK_REQUIRE((A.q_st | A.q_sh | A.k_st | A.k_sh | A.v_st | A.v_sh) % 8 == 0,
              "qik_rotary: strides must be multiples of 8 elements");
  int page_log2 = 0;
  if (paged) {
    QIK_REQUIRE(A.page > 0 && A.page <= 4096 && (A.page & (A.page - 1)) == 0 && A.pages > 0 && A.pages <= 0x7FFFFFFFll,
                "qik_rotary: page of %lld tokens (a power of two), %lld pages", (long long)A.page, (long long)A.pages);
    QIK_REQUIRE((A.kp_s0 | A.kp_sh | A.kp_ss | A.vp_s0 | A.vp_sh | A.vp_ss) % 8 == 0,
                "qik_rotary: page strides must be multiples of 8 elements");
    while ((1ll << page_log2) < A.page) ++page_log2;
  }
  RotaryDev d;
  d.q = static_cast<const uint16_t*>(A.q), d.k = static_cast<const uint16_t*>(A.k);
  d.v = static_cast<const uint16_t*>(A.v);
  d.q_out = static_cast<uint16_t*>(A.q_out), d.k_out = static_cast<uint16_t*>(A.k_out);
  d.v_out = static_cast<uint16_t*>(A.v_out);
  d.positions = A.positions, d.slots = A.slots, d.cos = A.cos, d.sin = A.sin, d.status = status;
  d.T = A.T, d.q_st = A.q_st, d.k_st = A.k_st, d.v_st = A.v_st, d.q_sh = A.q_sh, d.k_sh = A.k_sh, d.v_sh = A.v_sh;
  d.P = static_cast<int>(A.P), d.HQ = static_cast<int>(A.HQ), d.HK = static_cast<int>(A.HK);
  d.HV = paged ? d.HK : 0;
  d.D = static_cast<int>(A.D), d.rot = static_cast<int>(A.rot), d.page_log2 = page_log2;
  d.interleaved = (A.flags & QIK_ROTARY_INTERLEAVED) != 0;
  d.pos64 = (A.flags & QIK_ROTARY_POS64) != 0;
  d.slot64 = (A.flags & QIK_ROTARY_SLOT64) != 0;
  d.paged = paged;
  if (paged) {
    d.kp_s0 = A.kp_s0, d.kp_sh = A.kp_sh, d.kp_ss = A.kp_ss, d.vp_s0 = A.vp_s0, d.vp_sh = A.vp_sh, d.vp_ss = A.vp_ss;
    d.n_slots = A.pages * A.page;
  } else {  // k out [T, HK, D]: "page" 0, the token its place
    d.kp_s0 = 0, d.kp_sh = A.D, d.kp_ss = A.HK * A.D, d.vp_s0 = d.vp_sh = d.vp_ss = 0;
    d.n_slots = 0;
  }
  const int heads_per_task = 32 / (d.D / 16) * kRotarySteps;
  d.tasks_per_token = (d.HQ + d.HK + d.HV + heads_per_task - 1) / heads_per_task;
  const int64_t ctas = (A.T * d.tasks_per_token + kRotaryWarps - 1) / kRotaryWarps;
  QIK_REQUIRE(ctas <= 0x7FFFFFFFll, "qik_rotary: %lld tokens are too many", (long long)A.T);
  const dim3 grid(static_cast<unsigned>(ctas)), block(kRotaryWarps * 32);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f16 = (A.flags & QIK_ROTARY_F16) != 0;
  cudaError_t e;
  if (d.D == 64)
    e = f16 ? launch_kernel(rotary_kernel<true, 4>, grid, block, 0, st, true, d)
            : launch_kernel(rotary_kernel<false, 4>, grid, block, 0, st, true, d);
  else if (d.D == 128)
    e = f16 ? launch_kernel(rotary_kernel<true, 8>, grid, block, 0, st, true, d)
            : launch_kernel(rotary_kernel<false, 8>, grid, block, 0, st, true, d);
  else
    e = f16 ? launch_kernel(rotary_kernel<true, 16>, grid, block, 0, st, true, d)
            : launch_kernel(rotary_kernel<false, 16>, grid, block, 0, st, true, d);
  QIK_TRY_CUDA(e);
  return check_launch("rotary_kernel");
}
