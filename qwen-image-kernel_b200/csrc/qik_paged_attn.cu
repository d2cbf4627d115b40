// qik_paged_attn.cu -- attention of new tokens over a paged KV cache.
//
//   out[i] = sum_j p_ij v_j / sum_j p_ij,   p_ij = 2^((q_i . k_j) * scale * log2(e) - m_i)
//
// over the keys j of the row's sequence that it sees: j <= limit (its own place in the
// sequence; the last key when not causal), and with a window j > limit - window or
// j < sinks.  m_i is the running maximum of an online softmax; scores, maxima, sums and
// the output accumulate in fp32.  p is rounded to the tensors' type before p . v, the operand
// of the 16-bit matrix instructions: a relative error of 2^-8 in bf16 and 2^-11 in fp16 at
// most (there up to 2^-25 absolute below 2^-14), which averages over the keys; the sum uses
// the unrounded p.  A row that sees no key is 0.
//
// The `group` query heads that share a key head are packed as rows: row r of a (sequence,
// key head) is token r / group, head r % group, so each K/V tile is read once for the
// whole group.  Two kernels, chosen by the rows of a sequence:
//
//   paged_split_kernel (at most 64 rows: single tokens and short drafts).  Bound by HBM:
//   a K/V byte meets at most 64 rows.  Work is counted in (sequence, key head, 64-key
//   tile) units and cut into equal contiguous ranges, one for each resident CTA, so
//   ragged batches and a single long sequence fill the GPU alike; every CTA finds its
//   range from the lengths on the device (the host needs none of them, a captured graph
//   follows them).  A (sequence, head) that one CTA covers is finished there; pieces go
//   to a workspace and are joined by paged_join_kernel in a fixed order.  Two
//   TMA warps fill a ring of K and V tiles; 8 warps split the tiles, their keys and the
//   16-row groups between them and run mma.sync m16n8k16: tcgen05's 128-row tiles would be
//   50 to 99% padding here and the tensor pipe is not what bounds it.
//
//   paged_tile_kernel (more rows: chunks and prompts).  Bound by the tensor core: two
//   128-row query tiles on tcgen05 share every 128-key tile, as in qik_attn.cu.
//
// Pages are fetched by TMA through a 5-D map (columns, place, half, head, page): an index outside the
// pool reads zeros, so a bad page table cannot fault; it is reported in the status word.
// A masked key has p = 0, and 0 x NaN would still spread through the product.  V rows that no row
// of the tile sees (behind the last token, before the window) are zeroed in shared memory,
// whatever an unused place of a page holds.  Where a row's result is not finite and a key that
// it does not see, but other rows of its tile do, has infinities or NaN in V, the row is computed
// again from the keys that it sees (mend_row, a path that finite values never take): a row's
// result depends on what it sees alone.  The CTA's waits know of it (paged_wait).
#include <mutex>
#include <type_traits>

#include "qik_device.cuh"
#include "qik_host.h"

namespace qik {

struct PagedDev {
  const uint16_t *q, *k_pages, *v_pages;
  uint16_t* out;
  const int32_t *table, *lens, *starts;
  float* ws_o;        // partial outputs
  float2* ws_ml;      // their (maximum, sum) per row
  int4* ws_desc;      // each CTA's open unit
  int* status;
  int64_t q_st, q_sh, o_st, o_sh, table_st;
  int64_t kp_s0, kp_sh, kp_ss, vp_s0, vp_sh, vp_ss;  // page strides (mend_row; TMA has its maps)
  int B, T, HK, G, W, pages, page_log2, max_new;
  int window, sinks, min_share;
  float scale_log2;
  bool causal, unit_mode;
  int tile_tok;          // tile kernel: tokens of a 128-row query tile (128 / G)
  int hi_rows;           // split kernel: most rows (new tokens x group) of a sequence
};

struct Seq {
  int q0, n, kv;
};
__device__ __forceinline__ Seq seq_of(const PagedDev& a, int i) {
  Seq s;
  s.q0 = min(max(__ldg(a.starts + i), 0), a.T);
  s.n = min(max(__ldg(a.starts + i + 1), s.q0), a.T) - s.q0;
  s.kv = min(max(__ldg(a.lens + i), 0), a.W << a.page_log2);
  return s;
}
// Lengths that seq_of had to bring into range (one CTA looks at them all).
__device__ __forceinline__ void report_bad_lengths(const PagedDev& a) {
  for (int i = threadIdx.x; i < a.B; i += blockDim.x) {
    const int q0 = __ldg(a.starts + i), q1 = __ldg(a.starts + i + 1), kv = __ldg(a.lens + i);
    if (q0 < 0 || q1 < q0 || q1 > a.T || q1 - q0 > a.max_new || kv < 0 || kv > (a.W << a.page_log2))
      report_bad_index(a.status);
  }
}
// Last and first key of token j (without the sinks); last < 0: none.
__device__ __forceinline__ int last_key(const PagedDev& a, const Seq& s, int j) {
  return a.causal ? s.kv - s.n + j : s.kv - 1;
}
__device__ __forceinline__ int first_key(const PagedDev& a, int last) {
  return a.window > 0 ? max(0, last - a.window + 1) : 0;
}
// The key tiles that tokens [j0, j1) of a sequence need: `sink` tiles from 0, then
// tiles [t0, t0 + main).
struct Tiles {
  int lmin, lmax;  // keys [lmin, lmax] and [0, sinks) are seen by some row
  int sink, t0, main;
};
template <int TILE>
__device__ __forceinline__ Tiles tiles_of(const PagedDev& a, const Seq& s, int j0, int j1) {
  Tiles t;
  t.lmax = last_key(a, s, j1 - 1);
  t.lmin = first_key(a, max(last_key(a, s, j0), 0));
  if (t.lmax < 0) {
    t.sink = t.t0 = t.main = 0;
  } else {
    t.t0 = t.lmin / TILE;
    t.main = t.lmax / TILE + 1 - t.t0;
    t.sink = min((min(a.sinks, t.lmax + 1) + TILE - 1) / TILE, t.t0);
  }
  return t;
}
__device__ __forceinline__ int tile_at(const Tiles& t, int u) { return u < t.sink ? u : t.t0 + u - t.sink; }

template <bool F16>
__device__ __forceinline__ float to_float(uint32_t half) {
  return F16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(half))) : __uint_as_float(half << 16);
}
// Bounded wait (mbar_wait) whose limit starts again while warps of the CTA form rows again:
// flags[0] says that a wait gave up, flags[1] how many warps are in mend_row.  That takes as long as a
// row has keys, with the pipeline's other roles waiting.
__device__ __forceinline__ bool paged_wait(uint64_t* bar, uint32_t parity, volatile int* flags, int* status) {
  if (mbar_try_wait(bar, parity)) return true;
  uint64_t t0 = globaltimer();
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 0u) {
      if (flags[0]) return false;
      const uint64_t now = globaltimer();
      if (flags[1] > 0) t0 = now;
      if (now - t0 > QIK_WAIT_NS) {
        flags[0] = 1;
        if (status) atomicExch(status, QIK_DEV_TIMEOUT);
        return false;
      }
    }
  }
}

template <bool F16>
__device__ __forceinline__ float dot8(const uint4& x, const uint4& y, float s) {
  const uint32_t a[4] = {x.x, x.y, x.z, x.w}, b[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fmaf(to_float<F16>(a[i] & 0xFFFFu), to_float<F16>(b[i] & 0xFFFFu), s);
    s = fmaf(to_float<F16>(a[i] >> 16), to_float<F16>(b[i] >> 16), s);
  }
  return s;
}
// Columns of o that are not finite, as bits 2c and 2c + 1 of pair c; `nan_only`: that are NaN.
template <int NC>
__device__ __forceinline__ uint32_t odd_columns(const float (&o)[NC][2], bool nan_only) {
  uint32_t r = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (nan_only ? isnan(o[c][i]) : !isfinite(o[c][i])) r |= 1u << (2 * c + i);
  return r;
}
// A row whose sums o (NC pairs of columns, the first two at `col`, the next ones `step` columns on,
// in units of 2^m) are not all finite: a column in which some key of the tiles [u0, u1) that the
// row does not see, and that is not zeroed for all rows, has infinities or NaN in V is formed
// again, key by key, from those that the row sees.  Whatever else makes a sum infinite or NaN stays.
// The keys are taken from the last one down, until every such column is NaN: where NaN has spread
// over a sequence, a row sees it at its own place, and this ends after one key.  (A column of
// infinities goes through all of them.)
template <int D, bool F16, int TILE, int NC>
__device__ __noinline__ void mend_row(const PagedDev& a, float (&o)[NC][2], int col, int step, Tiles t, int u0, int u1,
                                     int seq, int h, int row, int hq, int last, int first, float m) {
  static_assert(NC <= 16, "columns as bits of a word");
  const uint32_t odd = odd_columns(o, false);
  if (!odd) return;
  const int32_t* table = a.table + static_cast<int64_t>(seq) * a.table_st;
  auto page_at = [&](int kv) -> int64_t {
    const int at = kv >> a.page_log2, id = at < a.W ? __ldg(table + at) : -1;
    return id < a.pages ? id : -1;
  };
  auto v_at = [&](int64_t page, int kv) {
    return reinterpret_cast<const uint32_t*>(a.v_pages + page * a.vp_s0 + h * a.vp_sh +
                                             (kv & ((1 << a.page_log2) - 1)) * a.vp_ss + col);
  };
  auto sees = [&](int kv) { return kv <= last && (kv >= first || kv < a.sinks); };
  uint32_t spoilt = 0;
#pragma unroll 1
  for (int u = u1 - 1; u >= u0 && spoilt != odd; --u) {
    const int kv0 = tile_at(t, u) * TILE;
    if (kv0 + TILE - 1 <= last && (kv0 >= first || kv0 + TILE - 1 < a.sinks)) continue;
#pragma unroll 1
    for (int kv = kv0; kv < kv0 + TILE && spoilt != odd; ++kv) {
      if (sees(kv) || kv > t.lmax || (kv < t.lmin && kv >= a.sinks)) continue;
      const int64_t page = page_at(kv);
      if (page < 0) continue;
      const uint32_t* v = v_at(page, kv);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint32_t w = __ldg(v + c * (step / 2));
        if (!isfinite(to_float<F16>(w & 0xFFFFu))) spoilt |= odd & (1u << (2 * c));
        if (!isfinite(to_float<F16>(w >> 16))) spoilt |= odd & (2u << (2 * c));
      }
    }
  }
  if (!spoilt) return;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (spoilt & (1u << (2 * c + i))) o[c][i] = 0.0f;
  const uint4* q = reinterpret_cast<const uint4*>(a.q + static_cast<int64_t>(row) * a.q_st + static_cast<int64_t>(hq) * a.q_sh);
  bool open = true;
#pragma unroll 1
  for (int u = u1 - 1; u >= u0 && open; --u) {
    const int kv0 = tile_at(t, u) * TILE;
#pragma unroll 1
    for (int kv = kv0 + TILE - 1; kv >= kv0 && open; --kv) {
      const int64_t page = sees(kv) ? page_at(kv) : -1;
      if (page < 0) continue;  // (a page outside the pool reads zeros: it adds nothing)
      const uint4* k = reinterpret_cast<const uint4*>(a.k_pages + page * a.kp_s0 + h * a.kp_sh +
                                                      (kv & ((1 << a.page_log2) - 1)) * a.kp_ss);
      float s = 0.0f;
#pragma unroll 1
      for (int d = 0; d < D / 8; ++d) s = dot8<F16>(__ldg(q + d), __ldg(k + d), s);
      const float p = ex2(fmaf(s, a.scale_log2, -m));
      const uint32_t* v = v_at(page, kv);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint32_t w = __ldg(v + c * (step / 2));
        if (spoilt & (1u << (2 * c))) o[c][0] = fmaf(p, to_float<F16>(w & 0xFFFFu), o[c][0]);
        if (spoilt & (2u << (2 * c))) o[c][1] = fmaf(p, to_float<F16>(w >> 16), o[c][1]);
      }
      open = (spoilt & ~odd_columns(o, true)) != 0;
    }
  }
}
// Calls mend() in the lanes of a whole warp whose row is `odd`; the CTA's waits know of it.
template <typename Mend>
__device__ __forceinline__ void mend_rows(volatile int* flags, bool odd, Mend mend) {
  if (!__any_sync(0xffffffffu, odd)) return;
  if ((threadIdx.x & 31) == 0) atomicAdd(const_cast<int*>(flags + 1), 1);
  if (odd) mend();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) atomicSub(const_cast<int*>(flags + 1), 1);
}

// ============================================================ few rows: split over keys
constexpr int kSplitTile = 64;

// MT: 16-row groups; TEAMS: sets of warps that take turns at the tiles.  Up to 16 rows the CTA is
// small and two share an SM, so that one loads while the other changes sequence (the 64 x 500
// to 12000 keys decode step: 219 us; one CTA of twice the warps and stages: 233 to 245).  With
// fewer short units than SMs nothing is there to share with: two teams halve the time from
// tile to tile (one token over 300 keys: 8.1 -> 7.1 us).
template <int D, int MT, int TEAMS>
struct SplitShape {
  static constexpr int kCtasPerSm = MT == 1 && TEAMS == 1 ? 2 : 1;
  static constexpr int kWarps = MT == 1 ? 4 * TEAMS : 8;
  static constexpr int kTeams = TEAMS;
  static constexpr int kGroups = kWarps / MT;                     // key groups, of all teams
  static constexpr int kKeys = kSplitTile * kTeams / kGroups;     // keys of a warp in a tile (and 16 rows)
  static constexpr int kThreads = (kWarps + 2) * 32;              // consumers, K and V producers
  static constexpr int kTileBytes = kSplitTile * D * 2;           // a K or V tile
  static constexpr int kStages = 6 / kCtasPerSm * (128 / D);
  static constexpr int kMergePitch = D + 4;
  static constexpr int kMerge = kStages * 2 * kTileBytes;
  static constexpr int kMl = kMerge + (kGroups - 1) * MT * 8 * kMergePitch * 4;
  static constexpr int kBar = kMl + kGroups * MT * 16 * 8;
  static constexpr int kBytes = kBar + 2 * kStages * 8 + 128 + 1024;
  static_assert(kBytes * kCtasPerSm + 1024 * kCtasPerSm <= 233472, "shared memory above an SM's 228 KB");
};

// Barrier of `threads` threads that tells all of them whether any had `p`.
__device__ __forceinline__ bool named_bar_any(uint32_t id, uint32_t threads, bool p) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(p)), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  return F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}

// Tiles of sequence i that this launch takes (0: none of its rows are its business).  A
// sequence whose rows see no key still has one tile, all of it masked: its rows are
// written as zeros.
__device__ __forceinline__ int split_tiles(const PagedDev& a, int i, Seq& s, Tiles& t) {
  s = seq_of(a, i);
  const int rows = s.n * a.G;
  if (rows == 0 || rows > a.hi_rows) return 0;
  t = tiles_of<kSplitTile>(a, s, 0, s.n);
  return max(1, t.sink + t.main);
}

// A CTA's walk over its range of the units: sequence by sequence, head by head.
struct Walk {
  Seq s;
  Tiles t;
  int i, h, at, nt;      // sequence, head, tile within the unit, the unit's tiles
  int left;              // tiles left in the range
};
__device__ __forceinline__ bool walk_open(const PagedDev& a, Walk& w) {  // the unit at (i, h); skips empty sequences
  while (w.i < a.B) {
    w.nt = split_tiles(a, w.i, w.s, w.t);
    if (w.nt > 0) return true;
    ++w.i;
    w.h = w.at = 0;
  }
  return false;
}
__device__ __forceinline__ bool walk_next(const PagedDev& a, Walk& w, int taken) {
  w.left -= taken;
  w.at += taken;
  if (w.left <= 0) return false;
  if (w.at < w.nt) return true;  // (the range ended inside the unit)
  w.at = 0;
  if (++w.h < a.HK) return true;
  w.h = 0;
  ++w.i;
  return walk_open(a, w);
}

template <int D, int MT, int TEAMS, bool F16>
__global__ void __launch_bounds__(SplitShape<D, MT, TEAMS>::kThreads, SplitShape<D, MT, TEAMS>::kCtasPerSm)
    paged_split_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                       const __grid_constant__ PagedDev a) {
  using Sh = SplitShape<D, MT, TEAMS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Sh::kBar);
  uint64_t* empty = full + Sh::kStages;
  volatile int* flags = reinterpret_cast<volatile int*>(empty + Sh::kStages);
  volatile int* scan = reinterpret_cast<volatile int*>(smem + Sh::kMerge);  // before the merge buffer is used
  volatile int* found = reinterpret_cast<volatile int*>(smem + Sh::kMl);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < Sh::kStages; ++s) {
      mbar_init(&full[s], 2);  // the K and the V producer
      mbar_init(&empty[s], Sh::kWarps / Sh::kTeams);
    }
    flags[0] = flags[1] = 0;
    found[0] = a.B;
    fence_mbar_init();
  }
  if (warp >= Sh::kWarps && lane == 0) tma_prefetch_desc(warp == Sh::kWarps ? &tm_k : &tm_v);
  pdl_wait();
  __syncthreads();
  if (blockIdx.x == 0) report_bad_lengths(a);

  // ---- this CTA's range of tiles
  Walk w;
  int share = 0;
  if (a.unit_mode) {
    w.i = blockIdx.x / a.HK;
    w.h = blockIdx.x % a.HK;
    w.at = 0;
    w.nt = split_tiles(a, w.i, w.s, w.t);
    w.left = w.nt;
  } else {
    Seq s;
    Tiles t;
    int mine = 0, sum = 0;
    for (int i = threadIdx.x; i < a.B; i += Sh::kThreads) {
      mine = split_tiles(a, i, s, t) * a.HK;
      sum += mine;
    }
    // what the threads before this one hold, and all of them
    auto scan_block = [&](int v, int& total) {
      int incl = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      if (lane == 31) scan[warp] = incl;
      __syncthreads();
      total = 0;
#pragma unroll
      for (int k = 0; k < Sh::kThreads / 32; ++k) {
        if (k == warp) incl += total;
        total += scan[k];
      }
      return incl - v;
    };
    int total, excl = scan_block(sum, total);
    share = max(a.min_share, static_cast<int>((static_cast<uint32_t>(total) + gridDim.x - 1) / gridDim.x));
    const long long begin = static_cast<long long>(share) * blockIdx.x;
    w.left = static_cast<int>(min(static_cast<long long>(share), total - begin));
    if (w.left > 0) {  // uniform over the CTA: find the sequence that holds tile `begin`
      const int want = static_cast<int>(begin);
      int base = 0;
      for (int i0 = 0; i0 < a.B; i0 += Sh::kThreads) {
        const int i = i0 + threadIdx.x;
        if (a.B > Sh::kThreads) {
          mine = i < a.B ? split_tiles(a, i, s, t) * a.HK : 0;
          __syncthreads();  // the last sums have been read
          excl = base + scan_block(mine, total);
          base += total;
        }
        if (mine > 0 && excl <= want && want < excl + mine) {
          const int nt = mine / a.HK, rest = want - excl;
          found[1] = rest / nt;
          found[2] = rest % nt;
          found[0] = i;
        }
        if (base > want) break;
      }
      __syncthreads();
      w.i = found[0];
      w.h = found[1];
      w.at = found[2];
      if (w.i < a.B) w.nt = split_tiles(a, w.i, w.s, w.t);
      else w.left = 0;
    }
    __syncthreads();  // `found` and `scan` lie in the merge buffers
    if (threadIdx.x == 0) a.ws_desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
  }
  if (w.left <= 0) {
    pdl_trigger();
    return;
  }

  auto k_ptr = [&](int s) { return smem + s * 2 * Sh::kTileBytes; };
  auto v_ptr = [&](int s) { return smem + s * 2 * Sh::kTileBytes + Sh::kTileBytes; };

  const int box_log2 = min(a.page_log2, 6);  // tokens of one TMA piece: a page's share of a tile
  static_assert(kSplitTile == 64, "pieces of 2^box_log2 tokens");
  if (warp >= Sh::kWarps) {
    // ------------------------------------------------------------ producers (K, V)
    const bool is_k = warp == Sh::kWarps;
    const CUtensorMap* tm = is_k ? &tm_k : &tm_v;
    const int pieces_log2 = 6 - box_log2, pieces = 1 << pieces_log2;
    const int piece = lane & (pieces - 1);
    const int run = 32 >> pieces_log2;  // tiles whose page numbers one load of the warp brings
    int stage = 0;
    uint32_t phase = 1;
    bool more = true, ok = true;
    while (more && ok) {
      const int count = min(w.nt - w.at, w.left);
      const int32_t* row = a.table + static_cast<int64_t>(w.i) * a.table_st;
      // lane's page number for its piece of tile u0 + lane / pieces: one load serves `run` tiles,
      // and the next is in flight while they are issued.  Behind the last token (or outside
      // the table) there is none, which reads as zeros like any page outside the pool
      auto page_of = [&](int u0) {
        const int u = u0 + (lane >> pieces_log2);
        if (u >= w.at + count || w.t.main == 0) return -1;
        const int key = tile_at(w.t, u) * kSplitTile + (piece << box_log2);
        const int p = key >> a.page_log2;
        if (key >= w.s.kv || p >= a.W) return -1;
        const int id = __ldg(row + p);
        if (id < 0 || id >= a.pages) report_bad_index(a.status);
        return id < a.pages ? id : -1;
      };
      int cur = 0, next = page_of(w.at);
      for (int u = w.at; u < w.at + count; ++u) {
        const int k = (u - w.at) & (run - 1);
        if (k == 0) {
          cur = next;
          next = page_of(u + run);
        }
        const int id = __shfl_sync(0xffffffffu, cur, (k << pieces_log2) + piece);
        if (!__all_sync(0xffffffffu, paged_wait(&empty[stage], phase, flags, a.status))) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[stage], Sh::kTileBytes);
        __syncwarp();
        if (lane < pieces)
          tma_load_5d((is_k ? k_ptr(stage) : v_ptr(stage)) + (piece << box_log2) * (D * 2), tm, 0,
                      (tile_at(w.t, u) * kSplitTile + (piece << box_log2)) & ((1 << a.page_log2) - 1), 0, w.h, id,
                      &full[stage]);
        if (++stage == Sh::kStages) stage = 0, phase ^= 1u;
      }
      more = walk_next(a, w, count);
    }
  } else {
    // ------------------------------------------------------------ consumers
    const int mt = warp % MT, kg = warp / MT;
    const int team = kg * Sh::kTeams / Sh::kGroups;  // the tiles that this warp takes: every kTeams-th
    const int key0 = kg % (Sh::kGroups / Sh::kTeams) * Sh::kKeys;  // its first key in them
    int turn = 0;
    const int g = lane >> 2, c2 = (lane & 3) * 2;
    // byte of the 16-byte chunk ch of a key in a tile: pieces of 2^box_log2 keys, each as halves of
    // 64 columns in 128-byte-swizzled rows (a 16-key block never crosses a piece)
    auto place = [&](int key, int ch) {
      const int in = key & ((1 << box_log2) - 1);
      return (key - in) * (D * 2) + ((ch >> 3) << (box_log2 + 7)) + in * 128 + (((ch & 7) ^ (key & 7)) << 4);
    };
    int stage = 0;
    uint32_t phase = 0;
    bool more = true, ok = true;
    while (more && ok) {
      const int count = min(w.nt - w.at, w.left);
      const int rows = w.s.n * a.G;
      const bool mine = mt * 16 < rows;
      // this lane's two rows: token, limits; q fragments straight from global memory
      int lim[2], low[2];
      uint32_t qf[D / 16][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = mt * 16 + g + 8 * x;
        const int j = r / a.G, hq = w.h * a.G + r % a.G;
        const bool valid = r < rows;
        lim[x] = valid ? last_key(a, w.s, j) : w.t.lmax;  // (rows behind the last are not stored)
        low[x] = first_key(a, lim[x]);
        const uint16_t* src = a.q + static_cast<int64_t>(w.s.q0 + j) * a.q_st + static_cast<int64_t>(hq) * a.q_sh + c2;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          qf[k][x] = valid ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 16)) : 0u;
          qf[k][x + 2] = valid ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 16 + 8)) : 0u;
        }
      }
      const int first_last = last_key(a, w.s, 0), last_first = first_key(a, w.t.lmax);
      float o[D / 8][4];
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[n][c] = 0.0f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

      for (int u = w.at; u < w.at + count; ++u) {
        const int kv0 = tile_at(w.t, u) * kSplitTile;
        if (Sh::kTeams > 1 && (turn++ & 1) != team) {
          if (++stage == Sh::kStages) stage = 0, phase ^= 1u;
          continue;
        }
        if (!__all_sync(0xffffffffu, paged_wait(&full[stage], phase, flags, a.status))) {
          ok = false;
          break;
        }
        if (mine) {
          const uint32_t kb = smem_u32(k_ptr(stage)), vb = smem_u32(v_ptr(stage));
          // V rows that no row sees (see the top of the file)
          const bool edge = kv0 + kSplitTile - 1 > w.t.lmax || (kv0 < w.t.lmin && kv0 + kSplitTile - 1 >= a.sinks);
          if (edge) {
            for (int x = lane; x < Sh::kKeys * (D / 8); x += 32) {
              const int key = key0 + x / (D / 8), ch = x % (D / 8), kv = kv0 + key;
              if (kv > w.t.lmax || (kv < w.t.lmin && kv >= a.sinks))
                *reinterpret_cast<uint4*>(v_ptr(stage) + place(key, ch)) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();  // before the next TMA write of this stage
            __syncwarp();
          }
          // S = Q K^T for kKeys keys: a 16-key block's fragments are loaded back to back (one
          // shared-memory latency a block), then multiplied in chains of D / 32 products
          float s[Sh::kKeys / 8][4];
#pragma unroll
          for (int n2 = 0; n2 < Sh::kKeys / 16; ++n2) {
            constexpr int kBatch = MT == 1 ? D / 16 : 4;
            float odd[2][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) s[2 * n2][c] = s[2 * n2 + 1][c] = odd[0][c] = odd[1][c] = 0.0f;
#pragma unroll
            for (int k0 = 0; k0 < D / 16; k0 += kBatch) {
              uint32_t kf[kBatch][4];
#pragma unroll
              for (int k = 0; k < kBatch; ++k) {
                const int key = key0 + n2 * 16 + (lane >> 4) * 8 + (lane & 7);
                ldsm4(kf[k], kb + place(key, (k0 + k) * 2 + ((lane >> 3) & 1)));
              }
#pragma unroll
              for (int k = 0; k < kBatch; k += 2) {
                mma16816<F16>(s[2 * n2], qf[k0 + k], kf[k][0], kf[k][1]);
                mma16816<F16>(s[2 * n2 + 1], qf[k0 + k], kf[k][2], kf[k][3]);
                mma16816<F16>(odd[0], qf[k0 + k + 1], kf[k + 1][0], kf[k + 1][1]);
                mma16816<F16>(odd[1], qf[k0 + k + 1], kf[k + 1][2], kf[k + 1][3]);
              }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) s[2 * n2][c] += odd[0][c], s[2 * n2 + 1][c] += odd[1][c];
          }
          // V fragments of the first 16 keys: in flight during the softmax
          uint32_t vf[D / 16][4];
          auto load_v = [&](int k2) {
#pragma unroll
            for (int d2 = 0; d2 < D / 16; ++d2) {
              const int key = key0 + k2 * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
              ldsm4_t(vf[d2], vb + place(key, d2 * 2 + (lane >> 4)));
            }
          };
          load_v(0);
          // masks, unless every row sees the whole tile
          const bool whole = kv0 + kSplitTile - 1 <= first_last && (kv0 >= last_first || kv0 + kSplitTile - 1 < a.sinks);
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int n = 0; n < Sh::kKeys / 8; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int x = c >> 1;
              s[n][c] *= a.scale_log2;
              if (!whole) {
                const int kv = kv0 + key0 + n * 8 + c2 + (c & 1);
                if (kv > lim[x] || (kv < low[x] && kv >= a.sinks)) s[n][c] = -INFINITY;
              }
              mx[x] = fmaxf(mx[x], s[n][c]);
            }
          float neg[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
            mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
            mx[x] = fmaxf(mx[x], m[x]);
          }
          if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
            float al[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              al[x] = mx[x] > m[x] ? ex2(m[x] - mx[x]) : 1.0f;  // 0 at the first seen key
              l[x] *= al[x];
              m[x] = mx[x];
            }
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
              for (int c = 0; c < 4; ++c) o[n][c] *= al[c >> 1];
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) neg[x] = m[x] == -INFINITY ? 0.0f : -m[x];
          uint32_t p[Sh::kKeys / 16][4];
#pragma unroll
          for (int n = 0; n < Sh::kKeys / 8; ++n) {
            float e[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              e[c] = ex2(s[n][c] + neg[c >> 1]);
              l[c >> 1] += e[c];
            }
            p[n >> 1][(n & 1) * 2] = pack16<F16>(e[0], e[1]);
            p[n >> 1][(n & 1) * 2 + 1] = pack16<F16>(e[2], e[3]);
          }
          // O += P V
#pragma unroll
          for (int k2 = 0; k2 < Sh::kKeys / 16; ++k2) {
            if (k2 > 0) load_v(k2);
#pragma unroll
            for (int d2 = 0; d2 < D / 16; ++d2) {
              mma16816<F16>(o[2 * d2], p[k2], vf[d2][0], vf[d2][1]);
              mma16816<F16>(o[2 * d2 + 1], p[k2], vf[d2][2], vf[d2][3]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
        if (++stage == Sh::kStages) stage = 0, phase ^= 1u;
      }
      // a wait that gave up ends the CTA's consumers together
      if (named_bar_any(1, Sh::kWarps * 32, !ok)) break;

      // ---- join the key groups: maxima and sums, then 8 of each 16 rows at a time; the first
      // group's warp adds the others' and stores
      float2* ml = reinterpret_cast<float2*>(smem + Sh::kMl);
      float* mg = reinterpret_cast<float*>(smem + Sh::kMerge);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        if ((lane & 3) == 0) ml[kg * MT * 16 + mt * 16 + g + 8 * x] = make_float2(m[x], l[x]);
      }
      named_bar_sync(1, Sh::kWarps * 32);
      const bool begins = w.at == 0, ends = w.at + count == w.nt;
      const int slot = 2 * blockIdx.x + (begins ? 1 : 0);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x == 1 && rows <= 8) break;
        const int r = mt * 16 + g + 8 * x;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int k = 0; k < Sh::kGroups; ++k) top = fmaxf(top, ml[k * MT * 16 + r].x);
#pragma unroll
        for (int k = 0; k < Sh::kGroups; ++k) {
          const float2 e = ml[k * MT * 16 + r];
          sum += e.x == -INFINITY ? e.y : e.y * ex2(e.x - top);  // (no key seen: 0, or NaN)
        }
        const float f = m[x] == -INFINITY ? 1.0f : ex2(m[x] - top);
        if (x == 1) named_bar_sync(1, Sh::kWarps * 32);
        float* part = mg + ((kg - 1) * MT * 8 + mt * 8 + g) * Sh::kMergePitch + c2;
        if (kg > 0) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(part + n * 8) = make_float2(o[n][2 * x] * f, o[n][2 * x + 1] * f);
        }
        named_bar_sync(1, Sh::kWarps * 32);
        if (kg == 0) {
          const float* src = mg + (mt * 8 + g) * Sh::kMergePitch + c2;
          const bool whole = begins && ends;
          const float inv = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
          const int64_t at = static_cast<int64_t>(slot) * (MT * 16) + r;
          uint16_t* dst = a.out + static_cast<int64_t>(w.s.q0 + r / a.G) * a.o_st +
                          static_cast<int64_t>(w.h * a.G + r % a.G) * a.o_sh + c2;
          float v[D / 8][2];
#pragma unroll
          for (int n = 0; n < D / 8; ++n) v[n][0] = o[n][2 * x] * f, v[n][1] = o[n][2 * x + 1] * f;
#pragma unroll
          for (int k = 0; k < Sh::kGroups - 1; ++k)
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
              const float2 e = *reinterpret_cast<const float2*>(src + k * MT * 8 * Sh::kMergePitch + n * 8);
              v[n][0] += e.x, v[n][1] += e.y;
            }
          if (w.s.n > 1)  // (one token: no row sees what another does not)
            mend_rows(flags, r < rows && odd_columns(v, false), [&] {
              float f[D / 8][2];
#pragma unroll
              for (int n = 0; n < D / 8; ++n) f[n][0] = v[n][0], f[n][1] = v[n][1];
              mend_row<D, F16, kSplitTile, D / 8>(a, f, c2, 8, w.t, w.at, w.at + count, w.i, w.h, w.s.q0 + r / a.G,
                                                  w.h * a.G + r % a.G, lim[x], low[x], top);
#pragma unroll
              for (int n = 0; n < D / 8; ++n) v[n][0] = f[n][0], v[n][1] = f[n][1];
            });
          if (r < rows && whole) {
#pragma unroll
            for (int n = 0; n < D / 8; ++n) *reinterpret_cast<uint32_t*>(dst + n * 8) = pack16<F16>(v[n][0] * inv, v[n][1] * inv);
          } else if (r < rows) {
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
              *reinterpret_cast<float2*>(a.ws_o + at * D + n * 8 + c2) = make_float2(v[n][0], v[n][1]);
          }
          if (r < rows && !whole && c2 == 0) a.ws_ml[at] = make_float2(top, sum);
        }
      }
      if (begins && !ends && threadIdx.x == 0)
        a.ws_desc[blockIdx.x] = make_int4(w.s.q0, w.h, static_cast<int>((w.nt - count + share - 1) / share), rows);
      more = walk_next(a, w, count);
    }
  }
  if (flags[0]) let_land();
  pdl_trigger();
}

// ============================================================ many rows: 128-row tiles
constexpr int kTileN = 128;                    // keys of a tile
constexpr int kTileM = 128;                    // rows of a query tile (one TMEM lane each)
constexpr int kTileRows = 2 * kTileM;          // rows of a CTA
constexpr int kTileSoftmaxWarps = 8;           // per query tile: two threads a row
constexpr int kTileThreads = 128 + 64 * kTileSoftmaxWarps;
constexpr float kTileRescale = 8.0f;           // O is rescaled when a maximum grows by > 2^8
constexpr int kTileSplitP = 2;                 // steps of 16 keys of each half of P handed over first (1, 3: 427 us)

__device__ __forceinline__ uint32_t bits_below(int n) {  // the lowest n bits, n clamped to [0, 32]
  return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u;
}

// One lane of the (whole) warp, the same at every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

template <int D>
struct TileShape {
  static constexpr int kHalves = D / 64;
  static constexpr int kHalfBytes = 128 * 128;             // 128 rows of 64 columns
  static constexpr int kOperand = kHalves * kHalfBytes;    // a 128-row tile of q, K or V
  static constexpr int kK0 = 2 * kOperand;
  static constexpr int kStages = 2;
  static constexpr int kV0 = kK0 + kStages * kOperand;
  static constexpr int kBar = kV0 + kStages * kOperand;
  static constexpr int kSeg = kBar + 512;                  // segment ring
  static constexpr int kBytes = kSeg + 4 * 80 + 1024;
  static_assert(kBytes <= 232448, "shared memory above the 227 KB per-CTA limit");
};

// A unit of this kernel is a (sequence, key head, block of two query tiles); its work is its key
// tiles and kUnitCost more for the change to it (first q and K, first softmax, last product and
// the stores: without it the CTAs with the many short units at a prompt's start end last).
constexpr int kUnitCost = 3;
struct Block {
  Seq s;
  Tiles t;
  int i, h, rb, blocks;  // sequence, key head, block, blocks of the sequence
  int at, nt;            // tile within the unit, the unit's tiles
  int taken;             // tiles of the unit that are in the CTA's range
  int left;              // work left in the CTA's range, this unit's not counted
};
__device__ __forceinline__ int row_blocks(const PagedDev& a, const Seq& s) {
  return (s.n + 2 * a.tile_tok - 1) / (2 * a.tile_tok);
}
__device__ __forceinline__ Tiles block_tiles(const PagedDev& a, const Seq& s, int rb) {
  const int j0 = rb * 2 * a.tile_tok;
  return tiles_of<kTileN>(a, s, j0, min(j0 + 2 * a.tile_tok, s.n));
}
// (a unit whose rows see no key still has one tile, so that its rows are written as zeros)
__device__ __forceinline__ int block_work(const PagedDev& a, const Seq& s, int rb) {
  const Tiles t = block_tiles(a, s, rb);
  return max(1, t.sink + t.main) + kUnitCost;
}
// Work of all row blocks of the sequence of one key head.  Whole warp: lanes with few
// blocks add theirs up alone, the others' blocks are shared out over the warp.
__device__ __forceinline__ int sequence_work(const PagedDev& a, const Seq& s, int blocks) {
  int sum = 0;
  if (blocks <= 4)
    for (int rb = 0; rb < blocks; ++rb) sum += block_work(a, s, rb);
  for (uint32_t big = __ballot_sync(0xffffffffu, blocks > 4); big; big &= big - 1) {
    const int l = __ffs(big) - 1;
    Seq o;
    o.q0 = 0;
    o.n = __shfl_sync(0xffffffffu, s.n, l);
    o.kv = __shfl_sync(0xffffffffu, s.kv, l);
    const int n = __shfl_sync(0xffffffffu, blocks, l);
    int part = 0;
    for (int rb = threadIdx.x & 31; rb < n; rb += 32) part += block_work(a, o, rb);
    part = __reduce_add_sync(0xffffffffu, part);
    if (static_cast<int>(threadIdx.x & 31) == l) sum = part;
  }
  return sum;
}
// Opens the unit at (i, h, rb) with `done` of its work (the change to it first, then its tiles) in
// earlier CTAs' ranges; false: the range ends before a tile of it.
__device__ __forceinline__ bool open_block(const PagedDev& a, Block& b, int done) {
  b.t = block_tiles(a, b.s, b.rb);
  b.nt = max(1, b.t.sink + b.t.main);
  b.at = max(0, done - kUnitCost);
  b.taken = min(b.nt, done + b.left - kUnitCost) - b.at;
  b.left -= b.nt + kUnitCost - done;
  return b.taken > 0;
}
__device__ __forceinline__ bool next_block(const PagedDev& a, Block& b) {
  if (b.left <= 0) return false;
  if (++b.rb == b.blocks) {
    b.rb = 0;
    if (++b.h == a.HK) {
      b.h = 0;
      do {
        if (++b.i >= a.B) return false;
        b.s = seq_of(a, b.i);
        b.blocks = row_blocks(a, b.s);
      } while (b.blocks == 0);
    }
  }
  return open_block(a, b, 0);
}
// The CTA's range of work: an equal share of all of it, counted sequence by sequence, head
// by head, row block by row block.  All threads; `slot`: 32 ints of shared memory.
__device__ __forceinline__ bool open_range(const PagedDev& a, Block& b, int& share, int* slot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  Seq s;
  if (a.unit_mode) {  // blockIdx.x: (sequence, block, head), the blocks of max_new tokens counted for all
    const int most = (a.max_new + 2 * a.tile_tok - 1) / (2 * a.tile_tok);
    b.h = blockIdx.x % a.HK;
    b.rb = blockIdx.x / a.HK % most;
    b.i = blockIdx.x / (a.HK * most);
    b.s = seq_of(a, b.i);
    b.blocks = row_blocks(a, b.s);
    if (b.rb >= b.blocks) return false;
    share = 1;
    b.left = 0x3FFFFFFF;
    open_block(a, b, 0);
    b.left = 0;
    return true;
  }
  int blocks, mine = 0, sum = 0;
  auto look = [&](int i) {
    s = seq_of(a, min(i, a.B - 1));
    blocks = i < a.B ? row_blocks(a, s) : 0;
    mine = sequence_work(a, s, blocks) * a.HK;
  };
  auto scan_block = [&](int v, int& total) {  // what the threads before this one hold, and all
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 31) slot[4 + warp] = incl;
    __syncthreads();
    int before = lane < warps ? slot[4 + lane] : 0;  // (a scan of the warps' sums by every warp)
    const int own = before;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += up;
    }
    total = __shfl_sync(0xffffffffu, before, 31);
    return incl - v + __shfl_sync(0xffffffffu, before - own, warp);
  };
  for (int i0 = 0; i0 < a.B; i0 += blockDim.x) {
    look(i0 + threadIdx.x);
    sum += mine;
  }
  int total, excl = scan_block(sum, total);
  share = max(a.min_share, static_cast<int>((static_cast<uint32_t>(total) + gridDim.x - 1) / gridDim.x));
  const long long begin = static_cast<long long>(share) * blockIdx.x;
  if (begin >= total) return false;
  const int want = static_cast<int>(begin);
  b.left = min(share, total - want);
  int base = 0;
  for (int i0 = 0; i0 < a.B; i0 += blockDim.x) {
    if (a.B > static_cast<int>(blockDim.x)) {
      look(i0 + threadIdx.x);
      excl = base + scan_block(mine, total);
      base += total;
    }
    if (mine > 0 && excl <= want && want < excl + mine) {
      slot[0] = i0 + threadIdx.x;
      slot[1] = (want - excl) / (mine / a.HK);
      slot[2] = (want - excl) % (mine / a.HK);
    }
    if (base > want) break;
  }
  __syncthreads();
  b.i = slot[0];
  b.h = slot[1];
  b.s = seq_of(a, b.i);
  b.blocks = row_blocks(a, b.s);
  int rest = slot[2];
  for (int rb0 = 0;; rb0 += 32) {  // the block that holds `rest` (every warp for itself)
    const int rb = rb0 + lane;
    const int work = rb < b.blocks ? block_work(a, b.s, rb) : 0;
    int incl = work;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, incl > rest);
    if (past) {
      const int l = __ffs(past) - 1;
      b.rb = rb0 + l;
      rest -= __shfl_sync(0xffffffffu, incl - work, l);
      break;
    }
    rest -= __shfl_sync(0xffffffffu, incl, 31);
    if (rb0 + 32 >= b.blocks) {  // (not reached: `rest` lies in the sequence)
      b.rb = b.blocks - 1;
      rest = 0;
      break;
    }
  }
  return open_block(a, b, rest);  // (uniform: the range may end before the unit's first tile)
}

// 32 of the D / 2 columns of O that each of a row's two threads has.
template <int D>
__device__ __forceinline__ void tmem_ld_cols(uint32_t addr, uint32_t (&r)[32]) {
  if constexpr (D == 128) tmem_ld_2x32(addr, r);
  else tmem_ld_2x32_at32(addr, r);
}
template <int D>
__device__ __forceinline__ void tmem_st_cols(uint32_t addr, const uint32_t (&r)[32]) {
  if constexpr (D == 128) tmem_st_2x32(addr, r);
  else tmem_st_2x32_at32(addr, r);
}

// Steps [FROM, TO) of 16 keys of a P half row: p = 2^(s * scale - m) of the thread's scores in pairs,
// packed over its own S columns; their fp32 sums are added to acc.  (2^x of some pairs on the
// FMA pipe, as qik_attn.cu does it, did not pay: the prompt of 8001 tokens took 417 us without, 421 with
// 9 of 32 pairs there, 428 with 13.)
template <bool F16, int FROM, int TO>
__device__ __forceinline__ void tile_softmax(const float (&sv)[64], float scale, float neg_m, uint32_t tP, uint64_t (&acc)[2]) {
  const uint64_t sc2 = f2_pack(scale, scale), nm2 = f2_pack(neg_m, neg_m);
#pragma unroll
  for (int i = FROM; i < TO; ++i) {
    uint32_t pk[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float x0, x1;
      f2_unpack(ffma2(f2_pack(sv[16 * i + 2 * j], sv[16 * i + 2 * j + 1]), sc2, nm2), x0, x1);
      const float p0 = ex2(x0), p1 = ex2(x1);
      acc[j & 1] = fadd2(acc[j & 1], f2_pack(p0, p1));
      pk[j] = pack16<F16>(p0, p1);
    }
    if (i == 0) __syncwarp();
    tmem_st_2x8(tP + 8 * i, pk);
  }
}

// What the warps know of a segment, in a ring in shared memory: kept there so that the softmax
// threads, which hold half a score row each, have their registers for that.
struct Segment {
  int valid, i, q0, h, tok0, toks;  // sequence, its first row of q, key head, new tokens of the block
  int n, n0, n1;                    // key tiles; of them, those that query tiles 0 and 1 need
  int kv0, sink_end, main0;         // first key; where the sink tiles end and the others begin
  int lmin, lmax, offset, kv;       // keys that some row sees; place of new token 0; tokens
  int begins, ends, pieces, pad;    // first / last segment of its unit; CTAs that follow with more of it
};
static_assert(sizeof(Segment) == 80, "segment ring");
constexpr int kSegRing = 4;

// One CTA per SM walks its range of the units' key tiles (open_range) segment by segment; a
// segment is a run of one unit's tiles.  All rings and barriers run on from segment to segment:
// the producer is ahead with the next segment's K and V while this one's last rows are stored.
//   warp 0      K and V tiles by TMA into 2-stage rings, V one tile behind K;
//   warp 1      MMA issuer (one elected lane): per tile t and query tile g, O_g += P_g(t) V_t, then
//               S_g(t + 1) = Q_g K_{t+1}^T (qik_attn.cu has the ordering argument);
//   warp 2      zeroes V rows that no row of the block sees;
//   warp 3      writes the segments; q by TMA, once the last segment's last S is done (a box is
//               (columns, group heads, tokens), which is the packed row order);
//   warps 4-19  softmax, eight warps per query tile, two threads a row.
// Query tile 0 ends earlier than tile 1 under a causal mask: its count of tiles is its own.
// A prompt of 8001 tokens with 24 heads of 128: 402 to 419 us by the clock, up to 977 TFLOP/s of the pairs that are seen; the tensor pipe
// and the special function unit are each 59% busy, the rest is the wait of a tile for its own product.
template <int D, bool F16>
__global__ void __launch_bounds__(kTileThreads, 1)
    paged_tile_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ PagedDev a) {
  using Sh = TileShape<D>;
  constexpr int kHalfO = D / 2;  // output columns of a softmax thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Sh::kBar);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;    // [2]
  uint64_t* k_empty = bars + 4;   // [2]
  uint64_t* v_full = bars + 6;    // [2] V ready for the product
  uint64_t* v_raw = bars + 8;     // [2] V landed, rows still to be zeroed
  uint64_t* v_empty = bars + 10;  // [2]
  uint64_t* s_full = bars + 12;   // [tile]
  uint64_t* p_full = bars + 14;   // [tile]
  uint64_t* o_full = bars + 16;   // [tile] the segment's last product is done
  uint64_t* o_empty = bars + 18;  // [tile] O has been read
  uint64_t* seg_full = bars + 20;   // [kSegRing]
  uint64_t* seg_empty = bars + 24;  // [kSegRing]
  uint64_t* h_full = bars + 28;   // [tile] the first 32 keys of each half of P
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 30);
  volatile int* flags = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* slot = reinterpret_cast<int*>(tmem_slot + 3);  // open_range: 4 + 20 words
  volatile Segment* ring = reinterpret_cast<volatile Segment*>(smem + Sh::kSeg);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_raw[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&h_full[s], kTileSoftmaxWarps);
      mbar_init(&p_full[s], kTileSoftmaxWarps);
      mbar_init(&o_full[s], 1);
      mbar_init(&o_empty[s], kTileSoftmaxWarps);
    }
    for (int s = 0; s < kSegRing; ++s) {
      mbar_init(&seg_full[s], 1);
      mbar_init(&seg_empty[s], 3 + 2 * kTileSoftmaxWarps);  // warps 0, 1 and 2, softmax
    }
    flags[0] = flags[1] = 0;
    fence_mbar_init();
  }
  pdl_wait();
  if (blockIdx.x == 0) report_bad_lengths(a);
  Block b;
  int share;
  const bool any = open_range(a, b, share, slot);
  if (threadIdx.x == 0 && !a.unit_mode) a.ws_desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (!any) {
    pdl_trigger();
    return;
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  uint8_t* sQ = smem;
  auto k_ptr = [&](int st) { return smem + Sh::kK0 + st * Sh::kOperand; };
  auto v_ptr = [&](int st) { return smem + Sh::kV0 + st * Sh::kOperand; };
  // segment number n of the CTA, or a segment that is not valid when a wait gave up
  auto seg_wait = [&](uint32_t n) -> bool {
    const bool ok = paged_wait(&seg_full[n & (kSegRing - 1)], (n / kSegRing) & 1, flags, a.status);
    return ok && ring[n & (kSegRing - 1)].valid;
  };
  auto kv_next = [](int kv0, int sink_end, int main0) { return kv0 + kTileN == sink_end ? main0 : kv0 + kTileN; };
  // V rows of the tile that no row of the block sees
  auto edge = [&](int kv0, int lmin, int lmax) {
    return kv0 + kTileN - 1 > lmax || (kv0 < lmin && kv0 + kTileN - 1 >= a.sinks);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    const int page = 1 << a.page_log2;
    const int box = min(page, kTileN);
    const int pieces = kTileN / box;
    uint32_t n_k = 0;  // tiles issued so far
    // the previous tile, whose V is still to be loaded
    int v_id = -1, v_place = 0, v_h = 0;
    bool v_owed = false, v_edge = false, ok = true;
    auto load = [&](const CUtensorMap* tm, uint8_t* dst, int id, int place, int h, uint64_t* bar) {
      if (lane == 0) mbar_arrive_expect_tx(bar, Sh::kOperand);
      __syncwarp();
      if (lane < pieces) {
#pragma unroll
        for (int hd = 0; hd < Sh::kHalves; ++hd)
          tma_load_5d(dst + hd * Sh::kHalfBytes + lane * box * 128, tm, 0, place, hd, h, id, bar);
      }
    };
    auto load_v = [&]() {  // V of the last tile issued, where it is still owed
      if (!v_owed) return;
      const int st = (n_k - 1) & 1;
      ok = ok && __all_sync(0xffffffffu, paged_wait(&v_empty[st], (((n_k - 1) >> 1) & 1) ^ 1u, flags, a.status));
      if (ok) load(&tm_v, v_ptr(st), v_id, v_place, v_h, v_edge ? &v_raw[st] : &v_full[st]);
      v_owed = false;
    };
    for (uint32_t seg = 0; ok && __all_sync(0xffffffffu, seg_wait(seg)); ++seg) {
      volatile Segment* sg = ring + (seg & (kSegRing - 1));
      const int n = sg->n, h = sg->h, kv = sg->kv, lmin = sg->lmin, lmax = sg->lmax, sink_end = sg->sink_end, main0 = sg->main0;
      int kv0 = sg->kv0;
      const int32_t* row = a.table + static_cast<int64_t>(sg->i) * a.table_st;
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[seg & (kSegRing - 1)]);
      // A segment without keys issues no K that V could follow, and with kSegRing - 1 of them in a row
      // the ring stays full until the softmax of the segment before them has its last V.
      if (n == 0) load_v();
      auto page_of = [&](int first) {
        if (lane >= pieces) return -1;
        const int key = first + lane * box;
        const int p = key >> a.page_log2;
        if (key >= kv || p >= a.W) return -1;
        const int id = __ldg(row + p);
        if (id < 0 || id >= a.pages) report_bad_index(a.status);
        return id < a.pages ? id : -1;
      };
      int next = n > 0 ? page_of(kv0) : -1;
      for (int t = 0; t < n && ok; ++t, ++n_k) {
        const int id = next, kv1 = kv_next(kv0, sink_end, main0);
        next = t + 1 < n ? page_of(kv1) : -1;
        const int st = n_k & 1, place = (kv0 + lane * box) & (page - 1);
        ok = __all_sync(0xffffffffu, paged_wait(&k_empty[st], ((n_k >> 1) & 1) ^ 1u, flags, a.status));
        if (!ok) break;
        load(&tm_k, k_ptr(st), id, place, h, &k_full[st]);
        load_v();
        v_owed = true;
        v_id = id, v_place = place, v_h = h, v_edge = edge(kv0, lmin, lmax);
        kv0 = kv1;
      }
    }
    if (ok) load_v();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp takes every step and one elected lane issues, from descriptors that are constants of
    // a stage: so they are warp-uniform values.  (One lane's branch around the loop, with descriptors
    // computed from the tile's number, was slower to issue than the tensor core to run them: the prompt of 8001
    // tokens took 460 us, 437 so.)
    constexpr uint32_t fmt = F16 ? 0 : 1;
    constexpr uint32_t idesc_s = idesc_f32acc(fmt, fmt, 0, 0, kTileM, kTileN);
    constexpr uint32_t idesc_o = idesc_f32acc(fmt, fmt, 0, 1, kTileM, D);
    const uint64_t q_desc = sdesc_sw128(smem_u32(sQ), 16, 1024);
    const uint64_t k_desc = sdesc_sw128(smem_u32(k_ptr(0)), 16, 1024);
    const uint64_t v_desc = sdesc_sw128(smem_u32(v_ptr(0)), Sh::kHalfBytes, 1024);
    constexpr uint64_t kOp16 = Sh::kOperand >> 4;
    uint32_t base = 0, q_n = 0, p_n[2] = {0u, 0u}, o_n[2] = {0u, 0u};  // tiles, q loads, P and O so far
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && __all_sync(0xffffffffu, paged_wait(bar, parity & 1u, flags, a.status));
    };
    auto commit = [&](uint64_t* bar) {
      if (elect_one()) umma_commit(bar);
      __syncwarp();
    };
    auto s_of = [&](int g, int st) {
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t off16 = ((i >> 2) * Sh::kHalfBytes + (i & 3) * 32) >> 4;
          umma_f16_ss(tmem + 128u * g, q_desc + g * kOp16 + off16, k_desc + st * kOp16 + off16, idesc_s, i > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[g]);
      }
      __syncwarp();
    };
    auto pv_of = [&](int g, int st, int part, bool first) {  // the steps of a part, of each half of P
      if (elect_one()) {
#pragma unroll
        for (int j = 0; j < kTileN / 16; ++j) {
          const int half = j / 4, i = j % 4;
          if ((i < kTileSplitP) != (part == 0)) continue;
          umma_f16_ts(tmem + 256u + 128u * g, tmem + 128u * g + 64u * half + 8u * i, v_desc + st * kOp16 + j * 128u, idesc_o,
                      !first || j > 0 ? 1u : 0u);
        }
      }
      __syncwarp();
    };
    auto issue_s = [&](int g, uint32_t k) {  // k: the CTA's tile
      if (k & 1) s_of(g, 1);
      else s_of(g, 0);
    };
    auto issue_pv = [&](int g, uint32_t k, int part, bool first) {
      if (k & 1) pv_of(g, 1, part, first);
      else pv_of(g, 0, part, first);
    };
    for (uint32_t seg = 0; ok && __all_sync(0xffffffffu, seg_wait(seg)); ++seg) {
      volatile Segment* sg = ring + (seg & (kSegRing - 1));
      const int n = sg->n, n0 = sg->n0, n1 = sg->n1, most = max(n0, n1);
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[seg & (kSegRing - 1)]);
      if (n == 0) continue;
      wait(q_full, q_n++);
      wait(&k_full[base & 1], base >> 1);
      tc_fence_after();
      if (ok) {
        if (n0 > 0) issue_s(0, base);
        if (n1 > 0) issue_s(1, base);
        commit(&k_empty[base & 1]);
        if (most <= 1) commit(q_empty);
      }
      for (int t = 0; t < n && ok; ++t) {
        const uint32_t k = base + t;
#pragma unroll
        for (int g = 0; g < 2; ++g) {  // (unrolled: p_n and o_n stay in registers)
          const int mine = g == 0 ? n0 : n1;
          if (ok && t < mine) {
            wait(&h_full[g], p_n[g]);
            if (g == 0 || n0 <= t) wait(&v_full[k & 1], k >> 1);
            if (t == 0 && o_n[g] > 0) wait(&o_empty[g], o_n[g] - 1);
            if (ok) {
              tc_fence_after();
              issue_pv(g, k, 0, t == 0);
              wait(&p_full[g], p_n[g]++);
            }
            if (ok) {
              tc_fence_after();
              issue_pv(g, k, 1, false);
              if (t == mine - 1) {
                commit(&o_full[g]);
                ++o_n[g];
              }
            }
          }
          if (g == 1 && ok) commit(&v_empty[k & 1]);
          if (ok && t + 1 < mine) {
            if (g == 0 || n0 <= t + 1) {
              wait(&k_full[(k + 1) & 1], (k + 1) >> 1);
              tc_fence_after();
            }
            if (ok) issue_s(g, k + 1);
          }
        }
        if (!ok) break;
        if (t + 1 < n) commit(&k_empty[(k + 1) & 1]);
        if (most > 1 && t + 2 == most) commit(q_empty);
      }
      base += n;
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ V rows nobody sees
    uint32_t base = 0, seen[2] = {0u, 0u};
    bool ok = true;
    for (uint32_t seg = 0; ok && __all_sync(0xffffffffu, seg_wait(seg)); ++seg) {
      volatile Segment* sg = ring + (seg & (kSegRing - 1));
      const int n = sg->n, lmin = sg->lmin, lmax = sg->lmax, sink_end = sg->sink_end, main0 = sg->main0;
      int kv0 = sg->kv0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[seg & (kSegRing - 1)]);
      for (int t = 0; t < n; ++t) {
        const int st = (base + t) & 1;
        if (edge(kv0, lmin, lmax)) {
          ok = __all_sync(0xffffffffu, paged_wait(&v_raw[st], seen[st]++ & 1u, flags, a.status));
          if (!ok) break;
          for (int key = lane >> 3; key < kTileN; key += 4) {
            const int kv = kv0 + key;
            if (kv > lmax || (kv < lmin && kv >= a.sinks)) {
#pragma unroll
              for (int hd = 0; hd < Sh::kHalves; ++hd)
                *reinterpret_cast<uint4*>(v_ptr(st) + hd * Sh::kHalfBytes + key * 128 + ((lane & 7) << 4)) =
                    make_uint4(0u, 0u, 0u, 0u);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_full[st]);
        }
        kv0 = kv_next(kv0, sink_end, main0);
      }
      base += n;
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------ segments and q
    if (lane == 0) {
      uint32_t q_n = 0;
      bool ok = true, more = true;
      for (uint32_t seg = 0; ok; ++seg) {
        volatile Segment* sg = ring + (seg & (kSegRing - 1));
        if (seg >= kSegRing) ok = paged_wait(&seg_empty[seg & (kSegRing - 1)], (seg / kSegRing - 1) & 1, flags, a.status);
        if (!ok) break;
        const int tok0 = b.rb * 2 * a.tile_tok, toks = min(b.s.n - tok0, 2 * a.tile_tok), n = b.t.main == 0 ? 0 : b.taken;
        sg->valid = more;
        if (more) {
          const int last = last_key(a, b.s, tok0 + min(toks, a.tile_tok) - 1);
          sg->i = b.i, sg->q0 = b.s.q0, sg->h = b.h, sg->tok0 = tok0, sg->toks = toks;
          sg->n = n;
          sg->n0 = last < 0 ? 0 : max(0, min(n, b.t.sink + last / kTileN - b.t.t0 + 1 - b.at));
          sg->n1 = toks > a.tile_tok ? n : 0;
          sg->kv0 = tile_at(b.t, b.at) * kTileN;
          sg->sink_end = b.t.sink > 0 ? b.t.sink * kTileN : -1;
          sg->main0 = b.t.t0 * kTileN;
          sg->lmin = b.t.lmin, sg->lmax = b.t.lmax, sg->kv = b.s.kv;
          sg->offset = b.s.kv - b.s.n;
          sg->begins = b.at == 0, sg->ends = b.at + b.taken == b.nt;
          sg->pieces = (b.nt - b.at - b.taken + share - 1) / share;
        }
        mbar_arrive(&seg_full[seg & (kSegRing - 1)]);
        if (!more) break;
        if (n > 0) {
          if (q_n > 0) ok = paged_wait(q_empty, (q_n - 1) & 1, flags, a.status);
          if (!ok) break;
          ++q_n;
          const int tiles = toks > a.tile_tok ? 2 : 1;
          mbar_arrive_expect_tx(q_full, tiles * Sh::kHalves * a.tile_tok * a.G * 128);
          for (int g = 0; g < tiles; ++g)
            for (int hd = 0; hd < Sh::kHalves; ++hd)
              tma_load_4d(sQ + g * Sh::kOperand + hd * Sh::kHalfBytes, &tm_q, 0, b.h * a.G, b.s.q0 + tok0 + g * a.tile_tok, hd, q_full);
        }
        more = next_block(a, b);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax (tile g)
    const int g = (warp - 4) >> 3;
    const int hc = lane >> 4;  // column half of the row
    // TMEM lane quarter warp % 4, its lower or upper 16 lanes by (warp / 4) % 2
    const int lane0 = (warp & 3) * 32 + (((warp - 4) >> 2) & 1) * 16;
    // the row's place in its query tile: token r / G of the tile, head r % G of the group; rows that
    // hold none (behind the last token, or the 128 % G last) follow another and are not stored
    const int r = lane0 + (lane & 15);
    const int tok = min(r / a.G, a.tile_tok - 1) + g * a.tile_tok;
    const uint32_t tS = tmem + (static_cast<uint32_t>(lane0) << 16) + 128u * g;
    const uint32_t tO = tS + 256u;
    uint32_t s_n = 0, o_n = 0;  // S tiles and segments of this query tile so far
    bool ok = true;
    for (uint32_t seg = 0; ok && __all_sync(0xffffffffu, seg_wait(seg)); ++seg) {
      volatile Segment* sg = ring + (seg & (kSegRing - 1));
      const int work = g == 0 ? sg->n0 : sg->n1;
      int my_last, my_first, kv0 = sg->kv0;
      {
        const int j = sg->tok0 + min(tok, sg->toks - 1);
        my_last = a.causal ? sg->offset + j : sg->kv - 1;
        my_first = first_key(a, my_last);
      }
      float m_run = -INFINITY, l_run = 0.0f;
      for (int t = 0; t < work; ++t, ++s_n) {
        if (!__all_sync(0xffffffffu, paged_wait(&s_full[g], s_n & 1, flags, a.status))) {
          ok = false;
          break;
        }
        tc_fence_after();
        float sv[64];
        {
          uint32_t rr[64];
          tmem_ld_2x64(tS, rr);
#pragma unroll
          for (int i = 0; i < 64; ++i) sv[i] = __uint_as_float(rr[i]);
        }
        const bool whole = __all_sync(0xffffffffu, kv0 + kTileN - 1 <= my_last &&
                                                       (kv0 >= my_first || kv0 + kTileN - 1 < a.sinks));
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (whole) {
#pragma unroll
          for (int c = 0; c < 64; c += 8) {
            mx[0] = fmaxf(fmaxf(mx[0], sv[c]), sv[c + 1]);
            mx[1] = fmaxf(fmaxf(mx[1], sv[c + 2]), sv[c + 3]);
            mx[2] = fmaxf(fmaxf(mx[2], sv[c + 4]), sv[c + 5]);
            mx[3] = fmaxf(fmaxf(mx[3], sv[c + 6]), sv[c + 7]);
          }
        } else {
          // seen columns as bits: below last + 1, and not below low or below sink
          const int col0 = kv0 + 64 * hc;
          uint32_t seen[2];
#pragma unroll
          for (int w = 0; w < 2; ++w)
            seen[w] = bits_below(my_last + 1 - col0 - 32 * w) &
                      (~bits_below(my_first - col0 - 32 * w) | bits_below(a.sinks - col0 - 32 * w));
#pragma unroll
          for (int c = 0; c < 64; ++c) {
            sv[c] = seen[c >> 5] & (1u << (c & 31)) ? sv[c] : -INFINITY;
            mx[c & 3] = fmaxf(mx[c & 3], sv[c]);
          }
        }
        // (NaN scores do not reach the maximum; they reach P and the sum)
        float raw_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        raw_max = fmaxf(raw_max, __shfl_xor_sync(0xffffffffu, raw_max, 16));
        const float tmax = raw_max * a.scale_log2;
        float alpha = 1.0f;
        bool rescale = false;
        if (tmax > m_run + kTileRescale || (m_run == -INFINITY && tmax > -INFINITY)) {
          rescale = m_run != -INFINITY;
          alpha = rescale ? ex2(m_run - tmax) : 0.0f;
          m_run = tmax;
        }
        const float neg_m = m_run == -INFINITY ? 0.0f : -m_run;
        uint64_t acc[2] = {0ull, 0ull};
        tile_softmax<F16, 0, kTileSplitP>(sv, a.scale_log2, neg_m, tS, acc);
        if (t >= 1 && __any_sync(0xffffffffu, rescale)) {
          const float f = rescale ? alpha : 1.0f;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            uint32_t rr[32];
            tmem_ld_cols<D>(tO + c * 32, rr);
#pragma unroll
            for (int i = 0; i < 32; ++i) rr[i] = __float_as_uint(__uint_as_float(rr[i]) * f);
            tmem_st_cols<D>(tO + c * 32, rr);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&h_full[g]);
        tile_softmax<F16, kTileSplitP, 4>(sv, a.scale_log2, neg_m, tS, acc);
        l_run = l_run * alpha + (f2_sum(acc[0]) + f2_sum(acc[1]));
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g]);
        kv0 = kv_next(kv0, sg->sink_end, sg->main0);
      }
      // ---- O / l, or this segment's piece of the unit
      const float l_row = l_run + __shfl_xor_sync(0xffffffffu, l_run, 16);
      if (work > 0 && ok) ok = __all_sync(0xffffffffu, paged_wait(&o_full[g], o_n++ & 1, flags, a.status));
      if (!ok) break;
      tc_fence_after();
      const bool stored = r < a.tile_tok * a.G && tok < sg->toks;
      const bool whole = sg->begins && sg->ends;
      const float inv = !whole ? 1.0f : l_row == 0.0f ? 0.0f : 1.0f / l_row;
      uint16_t* dst = a.out + static_cast<int64_t>(sg->q0 + sg->tok0 + tok) * a.o_st +
                      static_cast<int64_t>(sg->h * a.G + r % a.G) * a.o_sh + kHalfO * hc;
      const int64_t at = static_cast<int64_t>(2 * blockIdx.x + (sg->begins ? 1 : 0)) * kTileRows + g * kTileM + r;
#pragma unroll 1  // (code that a CTA runs a few times: fetching it is what it costs)
      for (int c = 0; c < D / 64; ++c) {
        uint32_t o[32];
        if (work > 0) {
          tmem_ld_cols<D>(tO + c * 32, o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (c == D / 64 - 1 && work > 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_empty[g]);
        }
        bool finite = true;
#pragma unroll
        for (int i = 0; i < 32; ++i) finite = finite && isfinite(__uint_as_float(o[i]));
        mend_rows(flags, !finite && stored && work > 0, [&] {
          // (the segment's tiles, counted as tile_at counts them)
          Tiles tl;
          tl.lmin = sg->lmin, tl.lmax = sg->lmax, tl.t0 = sg->main0 / kTileN, tl.main = 1;
          tl.sink = sg->sink_end > 0 ? sg->sink_end / kTileN : 0;
          const int k0 = sg->kv0 / kTileN, u0 = k0 < tl.sink ? k0 : k0 - tl.t0 + tl.sink;
          float f[16][2];
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i >> 1][i & 1] = __uint_as_float(o[i]);
          mend_row<D, F16, kTileN, 16>(a, f, kHalfO * hc + c * 32, 2, tl, u0, u0 + sg->n, sg->i, sg->h, sg->q0 + sg->tok0 + tok,
                                       sg->h * a.G + r % a.G, my_last, my_first, m_run);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(f[i >> 1][i & 1]);
        });
        if (stored && whole) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = pack16<F16>(__uint_as_float(o[i + 2 * k]) * inv, __uint_as_float(o[i + 2 * k + 1]) * inv);
            *reinterpret_cast<uint4*>(dst + c * 32 + i) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else if (stored) {
          uint4* part = reinterpret_cast<uint4*>(a.ws_o + at * D + kHalfO * hc + c * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i) part[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
      if (stored && !whole && hc == 0) a.ws_ml[at] = make_float2(m_run, l_row);
      if (warp == 4 && lane == 0 && sg->begins && !sg->ends) {
        a.ws_desc[blockIdx.x] = make_int4(sg->q0 + sg->tok0, sg->h, sg->pieces, sg->toks);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[seg & (kSegRing - 1)]);
    }
  }
  if (flags[0]) let_land();
  tc_fence_before();
  __syncthreads();
  pdl_trigger();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ============================================================ joining pieces
// out = sum_p f_p o_p / sum_p f_p l_p, f_p = 2^(m_p - max m), over the pieces of a unit that CTA
// `cta` left open: its own, then the following CTAs' first ones, added in that order.  One warp
// has kJoinRows rows; the first two pieces (mostly all there are) are loaded with their maxima.
// Small CTAs and few registers: this kernel is a chain of three memory latencies (the unit, its
// pieces, the stores) and is over sooner the more of its warps are resident.
constexpr int kJoinRows = 2;
constexpr int kJoinWarps = 2;

struct JoinDev {
  uint16_t* out;
  int64_t o_st, o_sh;
  const float* ws_o;
  const float2* ws_ml;
  const int4* ws_desc;
  int G, tile_tok, slot_rows;
  bool toks;  // the unit's rows are counted in query tiles of 128 (tile kernel)
};
// blockIdx.x: the kernel's CTAs; blockIdx.y: rows of the unit.
template <int D, bool F16>
__global__ void __launch_bounds__(kJoinWarps * 32, 12) paged_join_kernel(const JoinDev a) {
  using Vec = typename std::conditional<D == 128, float4, float2>::type;
  const int lane = threadIdx.x & 31, cta = blockIdx.x;
  const int r0 = (blockIdx.y * kJoinWarps + (threadIdx.x >> 5)) * kJoinRows;
  pdl_wait();
  const int4 d = __ldcg(a.ws_desc + cta);  // first row of q, head, further pieces, rows (tokens)
  uint16_t* dst[kJoinRows];
  bool any = false;
#pragma unroll
  for (int k = 0; k < kJoinRows; ++k) {
    const int r = r0 + k;
    const int in = a.toks ? r % kTileM : r, tok = a.toks ? in / a.G + r / kTileM * a.tile_tok : r / a.G;
    const bool mine = d.x >= 0 && (a.toks ? in < a.tile_tok * a.G && tok < d.w : r < d.w);
    any = any || mine;
    dst[k] = mine ? a.out + static_cast<int64_t>(d.x + tok) * a.o_st + static_cast<int64_t>(d.y * a.G + in % a.G) * a.o_sh : nullptr;
  }
  if (any) {
    const int pieces = 1 + d.z;
    auto at = [&](int p, int k) { return static_cast<int64_t>(p == 0 ? 2 * cta + 1 : 2 * (cta + p)) * a.slot_rows + r0 + k; };
    float2 ml[2][kJoinRows];
    Vec v[2][kJoinRows];
    float top[kJoinRows], sum[kJoinRows], acc[kJoinRows][D / 32];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int k = 0; k < kJoinRows; ++k) {
        ml[p][k] = __ldcg(a.ws_ml + at(p, k));
        v[p][k] = __ldcg(reinterpret_cast<const Vec*>(a.ws_o + at(p, k) * D) + lane);
      }
#pragma unroll
    for (int k = 0; k < kJoinRows; ++k) {
      top[k] = fmaxf(ml[0][k].x, ml[1][k].x);
      if (pieces > 2) {
        for (int p = 2 + lane; p < pieces; p += 32) top[k] = fmaxf(top[k], __ldcg(a.ws_ml + at(p, k)).x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));
      }
      sum[k] = 0.0f;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) acc[k][c] = 0.0f;
    }
    auto add = [&](int k, float2 e, const Vec& o) {
      const float f = e.x == -INFINITY ? (e.y == 0.0f ? 0.0f : 1.0f) : ex2(e.x - top[k]);  // (no key seen: 0, or NaN)
      sum[k] = fmaf(e.y, f, sum[k]);
      const float* x = reinterpret_cast<const float*>(&o);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) acc[k][c] = fmaf(x[c], f, acc[k][c]);
    };
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int k = 0; k < kJoinRows; ++k) add(k, ml[p][k], v[p][k]);
    for (int p0 = 2; p0 < pieces; p0 += 4) {  // (one long sequence: dozens of pieces)
      float2 more_ml[4][kJoinRows];
      Vec more_v[4][kJoinRows];
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int k = 0; k < kJoinRows; ++k)
          if (p0 + p < pieces) {
            more_ml[p][k] = __ldcg(a.ws_ml + at(p0 + p, k));
            more_v[p][k] = __ldcg(reinterpret_cast<const Vec*>(a.ws_o + at(p0 + p, k) * D) + lane);
          }
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int k = 0; k < kJoinRows; ++k)
          if (p0 + p < pieces) add(k, more_ml[p][k], more_v[p][k]);
    }
#pragma unroll
    for (int k = 0; k < kJoinRows; ++k) {
      const float inv = sum[k] == 0.0f ? 0.0f : 1.0f / sum[k];
      if (!dst[k]) continue;
      if constexpr (D == 128)
        reinterpret_cast<uint2*>(dst[k])[lane] = make_uint2(pack16<F16>(acc[k][0] * inv, acc[k][1] * inv),
                                                            pack16<F16>(acc[k][2] * inv, acc[k][3] * inv));
      else
        reinterpret_cast<uint32_t*>(dst[k])[lane] = pack16<F16>(acc[k][0] * inv, acc[k][1] * inv);
    }
  }
  pdl_trigger();
}

// ============================================================ host
constexpr int kSplitRows = 64;  // most rows of a sequence that the split kernel takes

struct PagedPlan {
  bool split;      // the split kernel, else the tile kernel
  bool unit_mode;  // one CTA a unit, nothing to join
  int mt, ctas, slot_rows, min_share, join_blocks;
  size_t o, ml, desc, bytes;  // workspace offsets
};

// Up to kSplitRows rows in every sequence: the split kernel; else the tile kernel for all of them (a
// single token among chunks still loads its keys at three quarters of the HBM rate there, and
// one kernel and its join are launched instead of two).  Short contexts are not cut: a join costs
// more than it gives (with units of at most 4 tiles instead of 8 left whole, the calls between
// took twice as long).  Shares have at least 4 tiles (split: 2 and 8 measured slower) or a unit's
// change and 2 (tile; 5 took 1% longer over 100 calls of mixed sizes, up to 23% on the small).
static PagedPlan paged_plan(const qik_paged_attn_args& A) {
  PagedPlan p = {};
  const int64_t G = A.HQ / A.HK, max_rows = A.max_new * G;
  const int sms = sm_count();
  p.split = max_rows <= kSplitRows;
  // the keys that a row can see bound the tiles of a unit
  const int64_t max_kv = A.max_kv < (1ll << 30) ? A.max_kv : 1ll << 30;  // (no page table holds more)
  const int64_t seen = A.window > 0 && A.window + A.max_new < max_kv ? A.window + A.max_new : max_kv;
  const int64_t sinks = A.window > 0 ? A.sinks : 0, size = p.split ? kSplitTile : kTileN;
  const int64_t tiles = (seen + size - 1) / size + (seen < max_kv ? 1 + (sinks + size - 1) / size : 0);
  int64_t units, work, rows = 0;
  if (p.split) {
    p.mt = max_rows <= 16 ? 1 : max_rows <= 32 ? 2 : 4;
    units = A.B * A.HK;
    work = units * tiles;
    // two teams of warps (mt 1 with units for at most the SMs) take a tile in 0.35 us, one in 0.65
    p.unit_mode = tiles <= 8 || (tiles <= 14 && (p.mt == 1 || units >= sms));
    p.ctas = sms * (p.mt == 1 ? 2 : 1);
    p.min_share = 4;
    p.slot_rows = p.mt * 16;
    rows = max_rows;
  } else {
    const int64_t block = 2 * (kTileM / G), by_rows = A.T / block + A.B, by_seq = A.B * ((A.max_new + block - 1) / block);
    units = (by_rows < by_seq ? by_rows : by_seq) * A.HK;
    work = units * (tiles + kUnitCost);
    p.unit_mode = tiles <= 8 && units <= 2 * sms && by_seq * A.HK <= 16 * sms;
    if (p.unit_mode) units = by_seq * A.HK;  // (counted without a look at the lengths)
    p.ctas = sms;
    p.min_share = kUnitCost + 2;
    p.slot_rows = kTileRows;
    rows = A.max_new <= block / 2 ? kTileM : kTileRows;
  }
  if (p.unit_mode) {
    p.ctas = static_cast<int>(units);
    return p;
  }
  // no more CTAs than there can be shares
  if ((work + p.min_share - 1) / p.min_share < p.ctas) p.ctas = static_cast<int>((work + p.min_share - 1) / p.min_share);
  p.join_blocks = static_cast<int>((rows + kJoinRows * kJoinWarps - 1) / (kJoinRows * kJoinWarps));
  auto take = [&](size_t bytes) {
    const size_t here = p.bytes;
    p.bytes += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t slots = static_cast<size_t>(2) * p.ctas * p.slot_rows;
  p.o = take(slots * A.D * sizeof(float));
  p.ml = take(slots * sizeof(float2));
  p.desc = take(p.ctas * sizeof(int4));
  return p;
}

static int check_paged(const qik_paged_attn_args& A) {
  QIK_REQUIRE(A.D == 64 || A.D == 128, "qik_paged_attention: head_dim %lld unsupported (64 or 128)", (long long)A.D);
  QIK_REQUIRE(A.B >= 0 && A.T >= 0 && A.HQ > 0 && A.HK > 0 && A.HQ % A.HK == 0 && A.HQ <= 65535 && A.B <= (1 << 20) &&
                  A.T <= 0x7FFFFFFFll && A.T * (A.HQ / A.HK) <= 0x7FFFFFFFll,
              "qik_paged_attention: bad sizes (%lld sequences, %lld tokens, %lld query and %lld key heads)",
              (long long)A.B, (long long)A.T, (long long)A.HQ, (long long)A.HK);
  QIK_REQUIRE(A.page >= 16 && A.page <= 4096 && (A.page & (A.page - 1)) == 0 && A.pages > 0 && A.pages <= 0x7FFFFFFFll,
              "qik_paged_attention: page of %lld tokens (a power of two, 16 to 4096), %lld pages", (long long)A.page,
              (long long)A.pages);
  QIK_REQUIRE(A.W >= 0 && A.W <= (1ll << 30) && A.W * A.page <= (1ll << 30), "qik_paged_attention: page table of %lld columns", (long long)A.W);
  // key tiles of all units are counted in 32 bits
  QIK_REQUIRE(A.HQ / A.HK <= 64, "qik_paged_attention: %lld query heads of one key head (64)", (long long)(A.HQ / A.HK));
  const int64_t blocks = A.T / (kTileM / (A.HQ / A.HK)) + A.B, keys = A.W * A.page;
  QIK_REQUIRE(blocks * A.HK <= 0x7FFFFFFFll && blocks * A.HK * (keys / kSplitTile + 3 + kUnitCost) <= 0x7FFFFFFFll,
              "qik_paged_attention: %lld tokens and %lld sequences of up to %lld keys are too much for one call", (long long)A.T,
              (long long)A.B, (long long)keys);
  QIK_REQUIRE(A.max_new >= 0 && A.max_new <= A.T && A.max_kv >= 0, "qik_paged_attention: max_new %lld of %lld tokens, max_kv %lld",
              (long long)A.max_new, (long long)A.T, (long long)A.max_kv);
  QIK_REQUIRE(A.window >= 0 && A.sinks >= 0 && A.window <= 0x3FFFFFFF && A.sinks <= 0x3FFFFFFF,
              "qik_paged_attention: window %d, sinks %d", A.window, A.sinks);
  QIK_REQUIRE(A.window == 0 || (A.flags & QIK_PAGED_CAUSAL), "qik_paged_attention: a window needs the causal form");
  QIK_REQUIRE(A.sm_scale > 0.0f && A.sm_scale < 1e30f, "qik_paged_attention: sm_scale must be positive and finite");
  return QIK_OK;
}

// (64 columns, place, 64-column half, head, page): one load brings a piece's halves one after
// the other; `halves` of them (the tile kernel's operands want them 128 rows apart and load
// them one by one).
static int page_map(CUtensorMap* m, const void* base, bool f16, const qik_paged_attn_args& A, int64_t s0, int64_t sh,
                    int64_t ss, int64_t tile, uint32_t halves) {
  const uint64_t dims[5] = {64, static_cast<uint64_t>(A.page), static_cast<uint64_t>(A.D / 64), static_cast<uint64_t>(A.HK),
                            static_cast<uint64_t>(A.pages)};
  const uint64_t strides[4] = {static_cast<uint64_t>(ss * 2), 128, static_cast<uint64_t>(sh * 2), static_cast<uint64_t>(s0 * 2)};
  const uint32_t box[5] = {64, static_cast<uint32_t>(A.page < tile ? A.page : tile), halves, 1, 1};
  return make_tmap_nd(m, base, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, dims,
                      strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Raise a kernel's shared-memory limit once per device.
template <typename K>
static cudaError_t allow_smem(K kernel, int bytes, std::once_flag* once) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&] { e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
  return e;
}

template <int D, int MT, int TEAMS, bool F16>
static cudaError_t launch_split(const CUtensorMap& tk, const CUtensorMap& tv, const PagedDev& d, int ctas, cudaStream_t st) {
  using Sh = SplitShape<D, MT, TEAMS>;
  static std::once_flag once[64];
  cudaError_t e = allow_smem(paged_split_kernel<D, MT, TEAMS, F16>, Sh::kBytes, once);
  if (e != cudaSuccess) return e;
  return launch_kernel(paged_split_kernel<D, MT, TEAMS, F16>, dim3(ctas), dim3(Sh::kThreads), Sh::kBytes, st, true, tk, tv, d);
}
template <int D, bool F16>
static cudaError_t launch_paged(const PagedPlan& p, PagedDev d, const CUtensorMap* maps, cudaStream_t st) {
  cudaError_t e;
  if (p.split) {
    const bool few = p.unit_mode && p.ctas <= sm_count();
    d.hi_rows = p.slot_rows;
    e = p.mt == 1   ? (few ? launch_split<D, 1, 2, F16>(maps[0], maps[1], d, p.ctas, st)
                           : launch_split<D, 1, 1, F16>(maps[0], maps[1], d, p.ctas, st))
        : p.mt == 2 ? launch_split<D, 2, 1, F16>(maps[0], maps[1], d, p.ctas, st)
                    : launch_split<D, 4, 1, F16>(maps[0], maps[1], d, p.ctas, st);
  } else {
    using Sh = TileShape<D>;
    static std::once_flag once[64];
    e = allow_smem(paged_tile_kernel<D, F16>, Sh::kBytes, once);
    if (e != cudaSuccess) return e;
    e = launch_kernel(paged_tile_kernel<D, F16>, dim3(p.ctas), dim3(kTileThreads), Sh::kBytes, st, true, maps[0], maps[1],
                      maps[2], d);
  }
  if (e != cudaSuccess || p.unit_mode) return e;
  const JoinDev j = {d.out, d.o_st, d.o_sh, d.ws_o, d.ws_ml, d.ws_desc, d.G, d.tile_tok, p.slot_rows, !p.split};
  return launch_kernel(paged_join_kernel<D, F16>, dim3(p.ctas, p.join_blocks), dim3(kJoinWarps * 32), 0,
                       st, true, j);
}

}  // namespace qik

using namespace qik;

extern "C" size_t qik_paged_attention_workspace_bytes(const qik_paged_attn_args* args) {
  if (!args || check_paged(*args) != QIK_OK || args->B == 0 || args->T == 0 || args->max_new == 0) return 0;
  return paged_plan(*args).bytes;
}

extern "C" int qik_paged_attention(const qik_paged_attn_args* args, void* ws, size_t ws_bytes, int* status, void* stream) {
  QIK_REQUIRE(args != nullptr, "qik_paged_attention: args is NULL");
  const qik_paged_attn_args& A = *args;
  int rc = check_paged(A);
  if (rc != QIK_OK) return rc;
  if (A.B == 0 || A.T == 0 || A.max_new == 0) return QIK_OK;
  QIK_REQUIRE(A.q && A.out && A.k_pages && A.v_pages && A.seq_lens && A.query_starts && (A.W == 0 || A.page_table),
              "qik_paged_attention: NULL pointer");
  QIK_REQUIRE(aligned16(A.q) && aligned16(A.out) && aligned16(A.k_pages) && aligned16(A.v_pages) && aligned16(ws),
              "qik_paged_attention: q, out, pages and workspace must be 16-byte aligned");
  QIK_REQUIRE((A.q_st | A.q_sh | A.o_st | A.o_sh | A.kp_s0 | A.kp_sh | A.kp_ss | A.vp_s0 | A.vp_sh | A.vp_ss) % 8 == 0 &&
                  A.q_st > 0 && A.q_sh > 0 && A.kp_s0 >= 0 && A.kp_sh >= 0 && A.kp_ss > 0 && A.vp_s0 >= 0 && A.vp_sh >= 0 && A.vp_ss > 0,
              "qik_paged_attention: strides must be multiples of 8 elements");
  const PagedPlan p = paged_plan(A);
  QIK_REQUIRE(p.bytes == 0 || (ws && ws_bytes >= p.bytes), "qik_paged_attention: workspace of %zu bytes, %zu needed",
              ws_bytes, p.bytes);
  const bool f16 = (A.flags & QIK_PAGED_F16) != 0;
  const int64_t tile = p.split ? kSplitTile : kTileN;
  const uint32_t halves = p.split ? static_cast<uint32_t>(A.D / 64) : 1;
  CUtensorMap maps[3];
  rc = page_map(&maps[0], A.k_pages, f16, A, A.kp_s0, A.kp_sh, A.kp_ss, tile, halves);
  if (!rc) rc = page_map(&maps[1], A.v_pages, f16, A, A.vp_s0, A.vp_sh, A.vp_ss, tile, halves);
  if (!rc && !p.split) {  // q: (64 columns, head, token, half), boxes of a group's heads and a query tile's tokens
    const uint64_t dims[4] = {64, static_cast<uint64_t>(A.HQ), static_cast<uint64_t>(A.T), static_cast<uint64_t>(A.D / 64)};
    const uint64_t strides[3] = {static_cast<uint64_t>(A.q_sh * 2), static_cast<uint64_t>(A.q_st * 2), 128};
    const uint32_t group = static_cast<uint32_t>(A.HQ / A.HK), box[4] = {64, group, kTileM / group, 1};
    rc = make_tmap_nd(&maps[2], A.q, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, dims, strides,
                      box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (rc) return rc;
  PagedDev d = {};
  d.q = static_cast<const uint16_t*>(A.q);
  d.out = static_cast<uint16_t*>(A.out);
  d.table = A.page_table, d.lens = A.seq_lens, d.starts = A.query_starts;
  d.status = status;
  d.k_pages = static_cast<const uint16_t*>(A.k_pages), d.v_pages = static_cast<const uint16_t*>(A.v_pages);
  d.kp_s0 = A.kp_s0, d.kp_sh = A.kp_sh, d.kp_ss = A.kp_ss, d.vp_s0 = A.vp_s0, d.vp_sh = A.vp_sh, d.vp_ss = A.vp_ss;
  d.q_st = A.q_st, d.q_sh = A.q_sh, d.o_st = A.o_st, d.o_sh = A.o_sh, d.table_st = A.table_st;
  d.B = static_cast<int>(A.B), d.T = static_cast<int>(A.T), d.HK = static_cast<int>(A.HK);
  d.G = static_cast<int>(A.HQ / A.HK), d.W = static_cast<int>(A.W), d.pages = static_cast<int>(A.pages);
  while ((1ll << d.page_log2) < A.page) ++d.page_log2;
  d.max_new = static_cast<int>(A.max_new);
  d.tile_tok = 128 / d.G;
  d.window = A.window, d.sinks = A.window > 0 ? A.sinks : 0;
  d.unit_mode = p.unit_mode, d.min_share = p.min_share;
  d.scale_log2 = A.sm_scale * 1.4426950408889634f;
  d.causal = (A.flags & QIK_PAGED_CAUSAL) != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* w = static_cast<uint8_t*>(ws);
  d.ws_o = reinterpret_cast<float*>(w + p.o);
  d.ws_ml = reinterpret_cast<float2*>(w + p.ml);
  d.ws_desc = reinterpret_cast<int4*>(w + p.desc);
  cudaError_t e = A.D == 128 ? (f16 ? launch_paged<128, true>(p, d, maps, st) : launch_paged<128, false>(p, d, maps, st))
                             : (f16 ? launch_paged<64, true>(p, d, maps, st) : launch_paged<64, false>(p, d, maps, st));
  QIK_TRY_CUDA(e);
  return check_launch("qik_paged_attention");
}
