// qik_norm.cu -- residual addition + RMS norm, with a 16-bit output or e4m3 codes and
// their scales.
//
//   h = x + r            (fp32; stored once, rounded to the tensors' type, as the new
//                         residual stream; r may be absent: h = x)
//   y = h * rsqrt(mean_cols(h^2) + eps) * w      (from the unrounded fp32 h)
//   plain:   y rounded once to the tensors' type
//   e4m3:    s = max(max|y| / 448, 1e-12) over the row or over the whole tensor,
//            codes = e4m3(y / s), nearest even; no 16-bit y exists in between
//
// Bound by HBM: 6 bytes an element in and out for h (x, r, h) and 1 or 2 for y.  A row
// is held in registers by one CTA between its load and its store, so a row's statistics
// cost no second read.  The whole-tensor scale needs every row's maximum before the
// first code: one kernel stores h, each row's 1 / rms and each CTA's max|y|, a second
// (its programmatic dependent) forms the same y from x and r again and packs it.
#include "qik_device.cuh"
#include "qik_host.h"

namespace qik {

// What the first kernel asks L2 to keep of x and r for the second (the last rows): 16 MB 74.1 us,
// 64 MB 71.3, 96 MB 71.0 at 8192 x 5120.
constexpr int64_t kNormKeepBytes = 64ll << 20;
constexpr int kNormMaxSlots = 2048;  // CTAs of the first kernel, each with one max|y|

struct NormDev {
  const void* x;
  const void* r;
  const void* w;
  void* h;
  void* y;           // 16-bit output (plain) or e4m3 codes
  float* scale;      // [M] (row scales) or [1]
  float* rstd;       // [M] workspace (whole-tensor scale)
  uint32_t* slots;   // [slot count] workspace: max|y| bits of each CTA of the first kernel
  int64_t M, ldx, ldr, keep_row;
  int N, n_slots;
  float eps;
};

enum NormMode { kNormPlain = 0, kNormRow = 1, kNormStats = 2 };

template <bool F16>
__device__ __forceinline__ void unpack8(const uint4 v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (F16) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    } else {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
}
template <bool F16>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = F16 ? pack_f16x2(f[2 * i], f[2 * i + 1]) : pack_bf16x2(f[2 * i], f[2 * i + 1]);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <bool F16, bool WF32>
__device__ __forceinline__ void load_weight8(const void* w, int vec, float (&f)[8]) {
  if (WF32) {
    const float4* p = reinterpret_cast<const float4*>(w) + 2 * static_cast<int64_t>(vec);
    const float4 a = __ldg(p), b = __ldg(p + 1);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    unpack8<F16>(__ldg(reinterpret_cast<const uint4*>(w) + vec), f);
  }
}
// A code takes the wrong side of a border when the quotient's error is larger than its distance
// from it, so max|y| / 448 and y / s are products with a rounded reciprocal that one step
// corrects to half a unit.  (Without it three times as many codes were off by a step; with f32x2
// arithmetic it costs nothing: 8192 x 5120 took 75.1 us before and 74.0 after.)
__device__ __forceinline__ float norm_scale(uint32_t amax_bits) {
  const float a = __uint_as_float(amax_bits), q = a * (1.0f / 448.0f), r = fmaf(-q, 448.0f, a);
  const float s = r == r ? fmaf(r, 1.0f / 448.0f, q) : q;  // infinity stays
  return s < 1e-12f ? 1e-12f : s;                          // NaN compares false and stays
}
struct Divisor {
  uint64_t s, inv;  // -s and 1 / s, each twice
};
// An infinite s divides every finite y to 0: its correction is made with 0 * inv.
__device__ __forceinline__ Divisor divisor(float s) {
  const float inv = __frcp_rn(s), d = inv == 0.0f ? 0.0f : -s;
  return {f2_pack(d, d), f2_pack(inv, inv)};
}
__device__ __forceinline__ uint2 codes8(const float (&y)[8], Divisor d) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t v = f2_pack(y[2 * i], y[2 * i + 1]), q = fmul2(v, d.inv);
    float a, b;
    f2_unpack(ffma2(ffma2(q, d.s, v), d.inv, q), a, b);
    o[i] = cvt_e4m3x2(a, b);
  }
  return make_uint2(o[0] | o[1] << 16, o[2] | o[3] << 16);
}
// |y| as bits: non-negative floats order like their bits, and NaN lies above infinity,
// so a maximum over bits lets a NaN through to the scale.
__device__ __forceinline__ uint32_t abs_bits(float y) { return __float_as_uint(y) & 0x7FFFFFFFu; }

// Block-wide sum (IsMax: maximum of bits) with one barrier: `buf` alternates between two
// halves from call to call, so a fast warp's next write cannot overtake a slow warp's read.
template <bool IsMax>
__device__ __forceinline__ uint32_t block_reduce(uint32_t v, uint32_t* buf) {
  const int warps = blockDim.x >> 5;
  if (IsMax) {
    v = __reduce_max_sync(0xffffffffu, v);
  } else {
    float f = __uint_as_float(v);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) f += __shfl_xor_sync(0xffffffffu, f, o);
    v = __float_as_uint(f);
  }
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t t = static_cast<int>(threadIdx.x & 31) < warps ? buf[threadIdx.x & 31] : 0u;
  if (IsMax) return __reduce_max_sync(0xffffffffu, t);
  float f = __uint_as_float(t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) f += __shfl_xor_sync(0xffffffffu, f, o);
  return __float_as_uint(f);
}

// One CTA walks rows blockIdx.x, + gridDim.x, ...; thread t holds the row's 8-element
// vectors t, t + blockDim.x, ... (VPT of them).
template <bool F16, bool WF32, int VPT, int MODE>
__global__ void __launch_bounds__(1024) add_rms_norm_kernel(const NormDev a) {
  __shared__ uint32_t red[4][32];
  const int nv = a.N >> 3;
  uint32_t top = 0;  // max|y| bits of every row this CTA walks (kNormStats)
  const uint64_t keep = l2_evict_last_policy(), pass = l2_evict_first_policy();
  pdl_wait();
  int turn = 0;
  uint4 xv[VPT], rv[VPT];
  auto load_row = [&](int64_t row) {
    const uint4* xr = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + row * a.ldx);
    const uint4* rr = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.r) + row * a.ldr);
    // the rows that the second kernel starts with stay in L2, the others leave it early
    const uint64_t pol = MODE == kNormStats && row >= a.keep_row ? keep : pass;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vec = threadIdx.x + j * blockDim.x;
      if (row < a.M && vec < nv) {
        xv[j] = ld_nc_hint(xr + vec, pol);
        if (a.r) rv[j] = ld_nc_hint(rr + vec, pol);
      }
    }
  };
#pragma unroll
  for (int j = 0; j < VPT; ++j) xv[j] = rv[j] = make_uint4(0u, 0u, 0u, 0u);
  load_row(blockIdx.x);
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x, turn ^= 1) {
    float h[VPT][8];
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vec = threadIdx.x + j * blockDim.x;
      unpack8<F16>(xv[j], h[j]);
      if (a.r) {
        float rf[8];
        unpack8<F16>(rv[j], rf);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[j][i] += rf[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(h[j][i], h[j][i], ss);
      if (a.h && vec < nv)
        __stcs(reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.h) + row * a.N) + vec, pack8<F16>(h[j]));
    }
    load_row(row + gridDim.x);  // in flight while this row is reduced and stored
    const float sum = __uint_as_float(block_reduce<false>(__float_as_uint(ss), red[turn]));
    const float rstd = rsqrtf(sum / static_cast<float>(a.N) + a.eps);
    if (MODE == kNormStats && threadIdx.x == 0) a.rstd[row] = rstd;
    uint32_t row_top = 0;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vec = threadIdx.x + j * blockDim.x;
      if (vec < nv) {
        float w[8];
        load_weight8<F16, WF32>(a.w, vec, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          h[j][i] = h[j][i] * rstd * w[i];
          if (MODE != kNormPlain) row_top = max(row_top, abs_bits(h[j][i]));
        }
        if (MODE == kNormPlain)
          reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.y) + row * a.N)[vec] = pack8<F16>(h[j]);
      }
    }
    if (MODE == kNormRow) {
      const float s = norm_scale(block_reduce<true>(row_top, red[2 + turn]));
      const Divisor inv = divisor(s);
      if (threadIdx.x == 0) a.scale[row] = s;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int vec = threadIdx.x + j * blockDim.x;
        if (vec < nv) reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.y) + row * a.N)[vec] = codes8(h[j], inv);
      }
    }
    if (MODE == kNormStats) top = max(top, row_top);
  }
  if (MODE == kNormStats) {
    const uint32_t m = block_reduce<true>(top, red[2]);
    if (threadIdx.x == 0) a.slots[blockIdx.x] = m;
  }
  pdl_trigger();
}

// The codes of a whole-tensor scale: y is formed again from x, r and the stored 1 / rms
// in the same order of operations (so max|y| is the value the scale came from).  Rows
// are walked from the last one up: the rows the first kernel read last are the ones
// still in L2.
template <bool F16, bool WF32, int VPT>
__global__ void __launch_bounds__(1024) rms_norm_codes_kernel(const NormDev a) {
  __shared__ uint32_t red[32];
  const int nv = a.N >> 3;
  const uint64_t pass = l2_evict_first_policy();
  pdl_wait();
  uint32_t m = 0;
  for (int i = threadIdx.x; i < a.n_slots; i += blockDim.x) m = max(m, __ldcg(a.slots + i));
  const float s = norm_scale(block_reduce<true>(m, red));
  const Divisor inv = divisor(s);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.scale = s;
  for (int64_t row = a.M - 1 - blockIdx.x; row >= 0; row -= gridDim.x) {
    const uint4* xr = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + row * a.ldx);
    const uint4* rr = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.r) + row * a.ldr);
    const float rstd = __ldcg(a.rstd + row);
    uint4 xv[VPT], rv[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vec = threadIdx.x + j * blockDim.x;
      xv[j] = rv[j] = make_uint4(0u, 0u, 0u, 0u);
      if (vec < nv) {
        xv[j] = ld_nc_hint(xr + vec, pass);
        if (a.r) rv[j] = ld_nc_hint(rr + vec, pass);
      }
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vec = threadIdx.x + j * blockDim.x;
      if (vec < nv) {
        float h[8], w[8];
        unpack8<F16>(xv[j], h);
        if (a.r) {
          float rf[8];
          unpack8<F16>(rv[j], rf);
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] += rf[i];
        }
        load_weight8<F16, WF32>(a.w, vec, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = h[i] * rstd * w[i];
        __stcs(reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.y) + row * a.N) + vec, codes8(h, inv));
      }
    }
  }
  pdl_trigger();
}

// Few rows (at most two for each CTA of one 8-CTA cluster) with a whole-tensor scale: the
// rows stay in registers while the CTAs exchange their max|y| through distributed shared
// memory, so one launch without a workspace does it.  Three rows of 4096: one launch and
// one allocation less on the host than the two kernels (which these sizes are bound by).
constexpr int kNormCluster = 8;
constexpr int kNormClusterRows = 2;
template <bool F16, bool WF32, int VPT>
__global__ void __launch_bounds__(1024) __cluster_dims__(kNormCluster, 1, 1) add_rms_norm_few_kernel(const NormDev a) {
  __shared__ uint32_t red[3][32];
  __shared__ uint32_t tops[kNormCluster];  // every CTA's max|y| bits, written by their owners
  const int nv = a.N >> 3;
  const uint32_t rank = cluster_ctarank();
  cluster_arrive_started();
  pdl_wait();
  float h[kNormClusterRows][VPT][8];
  uint4 xv[kNormClusterRows][VPT], rv[kNormClusterRows][VPT];
#pragma unroll
  for (int k = 0; k < kNormClusterRows; ++k) {
    const int64_t row = rank + k * kNormCluster;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vec = threadIdx.x + j * blockDim.x;
      xv[k][j] = rv[k][j] = make_uint4(0u, 0u, 0u, 0u);
      if (row < a.M && vec < nv) {
        xv[k][j] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + row * a.ldx) + vec);
        if (a.r) rv[k][j] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.r) + row * a.ldr) + vec);
      }
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < kNormClusterRows; ++k) {
    const int64_t row = rank + k * kNormCluster;
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vec = threadIdx.x + j * blockDim.x;
      unpack8<F16>(xv[k][j], h[k][j]);
      if (a.r) {
        float rf[8];
        unpack8<F16>(rv[k][j], rf);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[k][j][i] += rf[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(h[k][j][i], h[k][j][i], ss);
      if (a.h && row < a.M && vec < nv)
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.h) + row * a.N)[vec] = pack8<F16>(h[k][j]);
    }
    const float sum = __uint_as_float(block_reduce<false>(__float_as_uint(ss), red[k]));
    const float rstd = rsqrtf(sum / static_cast<float>(a.N) + a.eps);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vec = threadIdx.x + j * blockDim.x;
      if (row < a.M && vec < nv) {
        float w[8];
        load_weight8<F16, WF32>(a.w, vec, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          h[k][j][i] = h[k][j][i] * rstd * w[i];
          top = max(top, abs_bits(h[k][j][i]));
        }
      }
    }
  }
  top = block_reduce<true>(top, red[kNormClusterRows]);
  cluster_wait_started();  // (behind the loads: a CTA without rows gets here at once, ahead of its peers)
  if (threadIdx.x < kNormCluster) st_cluster_u32(mapa_shared(&tops[rank], threadIdx.x), top);
  cluster_sync();
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kNormCluster; ++i) m = max(m, tops[i]);
  const float s = norm_scale(m);
  const Divisor inv = divisor(s);
  if (rank == 0 && threadIdx.x == 0) *a.scale = s;
#pragma unroll
  for (int k = 0; k < kNormClusterRows; ++k) {
    const int64_t row = rank + k * kNormCluster;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int vec = threadIdx.x + j * blockDim.x;
      if (row < a.M && vec < nv)
        reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.y) + row * a.N)[vec] = codes8(h[k][j], inv);
    }
  }
  pdl_trigger();
}

struct NormShape {
  int threads, vpt;
};
// Two vectors a thread (four 16-byte loads in flight) up to 16384 columns, four above.
static NormShape norm_shape(int64_t N) {
  const int nv = static_cast<int>(N >> 3);
  NormShape s;
  s.vpt = nv <= 64 ? 1 : nv <= 2048 ? 2 : 4;
  s.threads = ((nv + s.vpt - 1) / s.vpt + 31) / 32 * 32;
  return s;
}
// As many CTAs as are resident at once (a second, partial wave of row walkers cost a third of
// the time at 8192 x 5120), evened out so that all walk the same number of rows or one less.
template <typename K>
static int norm_ctas(K kernel, int threads, int64_t M, int (&cache)[33]) {
  int& per_sm = cache[threads / 32];
  if (per_sm == 0) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != cudaSuccess || n < 1) n = 1;
    per_sm = n;
  }
  int64_t most = static_cast<int64_t>(sm_count()) * per_sm;
  if (most > kNormMaxSlots) most = kNormMaxSlots;
  if (M <= most) return static_cast<int>(M);
  const int64_t rows = (M + most - 1) / most;
  return static_cast<int>((M + rows - 1) / rows);
}

template <bool F16, bool WF32, int VPT>
static cudaError_t launch_norm(NormDev d, int mode, const NormShape& s, cudaStream_t st) {
  static int cache[4][33];
  const dim3 block(s.threads);
  switch (mode) {
    case kNormPlain: {
      auto k = add_rms_norm_kernel<F16, WF32, VPT, kNormPlain>;
      return launch_kernel(k, dim3(norm_ctas(k, s.threads, d.M, cache[0])), block, 0, st, true, d);
    }
    case kNormRow: {
      auto k = add_rms_norm_kernel<F16, WF32, VPT, kNormRow>;
      return launch_kernel(k, dim3(norm_ctas(k, s.threads, d.M, cache[1])), block, 0, st, true, d);
    }
    default: {
      if (VPT <= 2 && d.M <= kNormCluster * kNormClusterRows)
        return launch_kernel(add_rms_norm_few_kernel<F16, WF32, VPT <= 2 ? VPT : 2>, dim3(kNormCluster), block, 0, st, true, d);
      auto k = add_rms_norm_kernel<F16, WF32, VPT, kNormStats>;
      auto c = rms_norm_codes_kernel<F16, WF32, VPT>;
      d.n_slots = norm_ctas(k, s.threads, d.M, cache[2]);
      d.keep_row = d.M - kNormKeepBytes / (static_cast<int64_t>(d.N) * (d.r ? 4 : 2));
      cudaError_t e = launch_kernel(k, dim3(d.n_slots), block, 0, st, true, d);
      if (e != cudaSuccess) return e;
      return launch_kernel(c, dim3(norm_ctas(c, s.threads, d.M, cache[3])), block, 0, st, true, d);
    }
  }
}
template <bool F16, bool WF32>
static cudaError_t launch_norm_vpt(const NormDev& d, int mode, const NormShape& s, cudaStream_t st) {
  if (s.vpt == 1) return launch_norm<F16, WF32, 1>(d, mode, s, st);
  if (s.vpt == 2) return launch_norm<F16, WF32, 2>(d, mode, s, st);
  return launch_norm<F16, WF32, 4>(d, mode, s, st);
}

static int norm_entry(const char* who, const void* x, int64_t ldx, const void* r, int64_t ldr, const void* w,
                      int w_f32, int64_t M, int64_t N, float eps, int f16, void* h, void* y, float* scale, void* ws,
                      int mode, void* stream) {
  QIK_REQUIRE(M >= 0 && N > 0 && N % 8 == 0 && N <= 32768, "%s: %lld rows of %lld columns (a multiple of 8, at most 32768)",
              who, (long long)M, (long long)N);
  QIK_REQUIRE(eps >= 0.0f, "%s: eps must not be negative", who);
  if (M == 0) return QIK_OK;
  QIK_REQUIRE(x && w && y && (mode == kNormPlain || scale) && (mode != kNormStats || ws || M <= kNormCluster * kNormClusterRows && N <= 16384),
              "%s: NULL pointer", who);
  QIK_REQUIRE(aligned16(x) && aligned16(r) && aligned16(w) && aligned16(h) && aligned16(y) && aligned16(ws),
              "%s: pointers must be 16-byte aligned", who);
  QIK_REQUIRE(ldx >= N && ldx % 8 == 0 && (!r || (ldr >= N && ldr % 8 == 0)),
              "%s: row pitches must be multiples of 8 elements and hold a row", who);
  NormDev d = {};
  d.x = x, d.r = r, d.w = w, d.h = h, d.y = y, d.scale = scale;
  d.slots = static_cast<uint32_t*>(ws);
  d.rstd = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kNormMaxSlots * sizeof(uint32_t));
  d.M = M, d.ldx = ldx, d.ldr = ldr, d.N = static_cast<int>(N), d.eps = eps;
  const NormShape s = norm_shape(N);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  QIK_TRY_CUDA(f16 ? (w_f32 ? launch_norm_vpt<true, true>(d, mode, s, st) : launch_norm_vpt<true, false>(d, mode, s, st))
                   : (w_f32 ? launch_norm_vpt<false, true>(d, mode, s, st)
                            : launch_norm_vpt<false, false>(d, mode, s, st)));
  return check_launch(who);
}

}  // namespace qik

extern "C" size_t qik_add_rms_norm_workspace_bytes(int64_t M, int64_t N) {
  if (M <= qik::kNormCluster * qik::kNormClusterRows && N <= 16384) return 0;
  return qik::kNormMaxSlots * sizeof(uint32_t) + static_cast<size_t>(M) * sizeof(float);
}

extern "C" int qik_add_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                                int weight_f32, int64_t M, int64_t N, float eps, int f16, void* sum_out, void* out,
                                void* stream) {
  return qik::norm_entry("qik_add_rms_norm", x, ldx, residual, ldr, weight, weight_f32, M, N, eps, f16, sum_out, out,
                         nullptr, nullptr, qik::kNormPlain, stream);
}

extern "C" int qik_add_rms_norm_e4m3(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                                     int weight_f32, int64_t M, int64_t N, float eps, int f16, void* sum_out, void* q,
                                     float* scale, int row_scales, void* ws, void* stream) {
  return qik::norm_entry("qik_add_rms_norm_e4m3", x, ldx, residual, ldr, weight, weight_f32, M, N, eps, f16, sum_out,
                         q, scale, ws, row_scales ? qik::kNormRow : qik::kNormStats, stream);
}
