// qik_paged_attn.cu -- attention of new tokens over a paged KV cache.
//
//   out[i] = sum_j p_ij v_j / sum_j p_ij,   p_ij = 2^((q_i . k_j) * scale * log2(e) - m_i)
//
// over the keys j of the row's sequence that it sees: j <= limit (its own place in the
// sequence; the last key when not causal), and with a window j > limit - window or
// j < sinks.  m_i is the running maximum of an online softmax; scores, maxima, sums and
// the output accumulate in fp32, p is rounded to the tensors' type before p . v (its
// relative error, 2^-9 in bf16 and 2^-12 in fp16 at most, averages over the keys, and the
// sum uses the unrounded p).  A row that sees no key is 0.
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
//   to a workspace and are joined by paged_split_join_kernel in a fixed order.  Two
//   TMA warps fill a ring of K and V tiles; 8 warps split the tiles, their keys and the
//   16-row groups between them and run mma.sync m16n8k16: tcgen05's 128-row tiles would be
//   8 to 87% padding here and the tensor pipe is not what bounds it.
//
//   paged_tile_kernel (more rows: chunks and prompts).  Bound by the tensor core: two
//   128-row query tiles on tcgen05 share every 128-key tile, as in qik_attn.cu.
//
// Pages are fetched by TMA through a 5-D map (columns, place, half, head, page): an index outside the
// pool reads zeros, so a bad page table cannot fault; it is reported in the status word.
// V rows that no row of the tile sees (behind the last token, before the window) are
// zeroed in shared memory before the product: whatever an unused place of a page holds,
// NaN too, meets p = 0 there and would spread otherwise.
#include <mutex>
#include <type_traits>

#include "qik_device.cuh"
#include "qik_host.h"

namespace qik {

struct PagedDev {
  const uint16_t* q;
  uint16_t* out;
  const int32_t *table, *lens, *starts;
  float* ws_o;        // partial outputs
  float2* ws_ml;      // their (maximum, sum) per row
  int4* ws_desc;      // split kernel: each CTA's open unit
  int* status;
  int64_t q_st, q_sh, o_st, o_sh, table_st;
  int B, T, HK, G, W, pages, page_log2, max_new;
  int window, sinks, splits, min_share;
  float scale_log2;
  bool causal, unit_mode;
  int lo_rows, hi_rows;  // rows (new tokens x group) of the sequences this launch takes
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
    if ((q0 < 0 || q1 < q0 || q1 > a.T || q1 - q0 > a.max_new || kv < 0 || kv > (a.W << a.page_log2)) && a.status)
      atomicExch(a.status, QIK_DEV_BAD_INDEX);
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
  if (rows <= a.lo_rows || rows > a.hi_rows) return 0;
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
                       const PagedDev a) {
  using Sh = SplitShape<D, MT, TEAMS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Sh::kBar);
  uint64_t* empty = full + Sh::kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + Sh::kStages);
  volatile int* scan = reinterpret_cast<volatile int*>(smem + Sh::kMerge);  // before the merge buffer is used
  volatile int* found = reinterpret_cast<volatile int*>(smem + Sh::kMl);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < Sh::kStages; ++s) {
      mbar_init(&full[s], 2);  // the K and the V producer
      mbar_init(&empty[s], Sh::kWarps / Sh::kTeams);
    }
    *abort_flag = 0;
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
        if ((id < 0 || id >= a.pages) && a.status) atomicExch(a.status, QIK_DEV_BAD_INDEX);
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
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[stage], phase, abort_flag, a.status))) {
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
        if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, abort_flag, a.status))) {
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
  pdl_trigger();
}

// sum_p f_p o_p / sum_p f_p l_p, f_p = 2^(m_p - max m), over the pieces of one row: `at(p)` is
// piece p's row in the workspace.  One warp; lane holds D / 32 columns.  Pieces are added in
// order, four loads in flight.
template <int D, bool F16, typename At>
__device__ __forceinline__ void join_row(const PagedDev& a, int pieces, At at, uint16_t* dst) {
  using Vec = typename std::conditional<D == 128, float4, float2>::type;
  const int lane = threadIdx.x & 31;
  float top = -INFINITY, sum = 0.0f;
  for (int p = lane; p < pieces; p += 32) top = fmaxf(top, __ldcg(a.ws_ml + at(p)).x);
  float acc[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) acc[c] = 0.0f;
  for (int p0 = 0; p0 < pieces; p0 += 4) {
    float2 ml[4];
    Vec v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t row = at(min(p0 + k, pieces - 1));
      ml[k] = __ldcg(a.ws_ml + row);
      v[k] = __ldcg(reinterpret_cast<const Vec*>(a.ws_o + row * D) + lane);
    }
    if (p0 == 0) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = p0 + k >= pieces || ml[k].x == -INFINITY ? 0.0f : ex2(ml[k].x - top);
      if (p0 + k < pieces) {
        sum = fmaf(ml[k].y, f, sum);
        const float* e = reinterpret_cast<const float*>(&v[k]);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) acc[c] = fmaf(e[c], f, acc[c]);
      }
    }
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  if constexpr (D == 128)
    reinterpret_cast<uint2*>(dst)[lane] =
        make_uint2(pack16<F16>(acc[0] * inv, acc[1] * inv), pack16<F16>(acc[2] * inv, acc[3] * inv));
  else
    reinterpret_cast<uint32_t*>(dst)[lane] = pack16<F16>(acc[0] * inv, acc[1] * inv);
}

// Joins the pieces of the unit that CTA blockIdx.x of the split kernel left open: its own
// piece, then the following CTAs' first pieces.  Four rows a CTA.
template <int D, bool F16>
__global__ void __launch_bounds__(128) paged_split_join_kernel(const PagedDev a, int slot_rows) {
  pdl_wait();
  const int4 d = __ldcg(a.ws_desc + blockIdx.x);  // first new token, head, further pieces, rows
  const int r = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (d.x >= 0 && r < d.w)
    join_row<D, F16>(a, 1 + d.z, [&](int p) {
      return static_cast<int64_t>(p == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + p)) * slot_rows + r;
    }, a.out + static_cast<int64_t>(d.x + r / a.G) * a.o_st + static_cast<int64_t>(d.y * a.G + r % a.G) * a.o_sh);
  pdl_trigger();
}

// ============================================================ many rows: 128-row tiles
constexpr int kTileN = 128;                    // keys of a tile
constexpr int kTileM = 128;                    // rows of a query tile (one TMEM lane each)
constexpr int kTileRows = 2 * kTileM;          // rows of a CTA
constexpr int kTileSoftmaxWarps = 8;           // per query tile: two threads a row
constexpr int kTileThreads = 128 + 64 * kTileSoftmaxWarps;
constexpr int kTileLoadWarps = kTileThreads / 32 - 2;  // warps that load q
constexpr float kTileRescale = 8.0f;           // O is rescaled when a maximum grows by > 2^8
constexpr int kTilePolyFrom = 23;              // pairs of a half row from here on take 2^x on the FMA pipe

__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {  // NaN if any is
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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
  static constexpr int kBytes = kBar + 256 + 1024;
  static_assert(kBytes <= 232448, "shared memory above the 227 KB per-CTA limit");
};

// Which sequence and which 256-row block of it a CTA has: blocks are counted over the
// sequences that this launch takes.  All threads; `slot` in shared memory.
__device__ __forceinline__ bool find_block(const PagedDev& a, int block, int* slot, int warps) {
  // slot[0..1]: sequence, row block; slot[2 ..]: warp sums
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) slot[0] = -1;
  int base = 0;
  for (int i0 = 0; i0 < a.B; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    int mine = 0;
    if (i < a.B) {
      const int rows = seq_of(a, i).n * a.G;
      if (rows > a.lo_rows && rows <= a.hi_rows) mine = (rows + kTileRows - 1) / kTileRows;
    }
    int incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 31) slot[2 + warp] = incl;
    __syncthreads();
    for (int k = 0; k < warp; ++k) incl += slot[2 + k];
    const int excl = base + incl - mine;
    if (mine > 0 && excl <= block && block < excl + mine) {
      slot[0] = i;
      slot[1] = block - excl;
    }
    for (int k = 0; k < warps; ++k) base += slot[2 + k];
    if (base > block) break;
  }
  __syncthreads();
  return slot[0] >= 0;
}

// TMEM accesses of half a row of D columns by each of a row's two threads.
template <int D>
__device__ __forceinline__ void tmem_ld_half(uint32_t addr, uint32_t (&r)[D / 2]) {
  if constexpr (D == 128) tmem_ld_2x64(addr, r);
  else tmem_ld_2x32_at32(addr, r);
}
template <int D>
__device__ __forceinline__ void tmem_st_half(uint32_t addr, const uint32_t (&r)[D / 2]) {
  if constexpr (D == 128) {
    uint32_t lo[32], hi[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) lo[i] = r[i], hi[i] = r[32 + i];
    tmem_st_2x32(addr, lo);
    tmem_st_2x32(addr + 32, hi);
  } else {
    tmem_st_2x32_at32(addr, r);
  }
}

// P half row: the thread's 64 scores, p = 2^(s * scale - m) in pairs, packed over its own
// S columns (as qik_attn.cu's softmax_half_row); returns the half row's fp32 sum.
template <bool kPoly, bool F16>
__device__ __forceinline__ float tile_softmax(const float (&sv)[64], float scale, float neg_m, uint32_t tP) {
  const uint64_t sc2 = f2_pack(scale, scale), nm2 = f2_pack(neg_m, neg_m);
  uint64_t acc[2] = {0ull, 0ull};
  uint32_t pk[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const uint64_t x2 = ffma2(f2_pack(sv[2 * j], sv[2 * j + 1]), sc2, nm2);
    uint64_t p2;
    if (kPoly && j >= kTilePolyFrom) {
      p2 = exp2_poly2(x2);
    } else {
      float x0, x1;
      f2_unpack(x2, x0, x1);
      p2 = f2_pack(ex2(x0), ex2(x1));
    }
    acc[j & 1] = fadd2(acc[j & 1], p2);
    float p0, p1;
    f2_unpack(p2, p0, p1);
    pk[j] = pack16<F16>(p0, p1);
  }
  __syncwarp();
  tmem_st_2x32(tP, pk);
  return f2_sum(acc[0]) + f2_sum(acc[1]);
}

template <int D, bool F16>
__global__ void __launch_bounds__(kTileThreads, 1)
    paged_tile_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const PagedDev a) {
  using Sh = TileShape<D>;
  constexpr int kHalfO = D / 2;  // output columns of a softmax thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Sh::kBar);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;    // [2]
  uint64_t* k_empty = bars + 3;   // [2]
  uint64_t* v_full = bars + 5;    // [2] V ready for the product
  uint64_t* v_raw = bars + 7;     // [2] V landed, rows still to be zeroed
  uint64_t* v_empty = bars + 9;   // [2]
  uint64_t* s_full = bars + 11;   // [tile]
  uint64_t* p_full = bars + 13;   // [tile]
  uint64_t* o_full = bars + 15;   // [tile]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 17);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* slot = reinterpret_cast<int*>(tmem_slot + 2);  // find_block: 2 + 20 words

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // heaviest first: under causal masks the last blocks of a sequence see the most keys
  const int block = static_cast<int>(gridDim.y - 1 - blockIdx.y);
  const int h = blockIdx.x;

  if (threadIdx.x == 0) {
    mbar_init(q_full, kTileLoadWarps);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_raw[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], kTileSoftmaxWarps);
      mbar_init(&o_full[s], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  pdl_wait();
  __syncthreads();
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) report_bad_lengths(a);
  if (!find_block(a, block, slot, kTileThreads / 32)) {
    pdl_trigger();
    return;
  }
  const int seq = slot[0];
  const int row0 = slot[1] * kTileRows;  // first packed row of this CTA
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Seq s = seq_of(a, seq);
  const int rows = min(s.n * a.G - row0, kTileRows);
  const int n_q = rows > kTileM ? 2 : 1;  // query tiles with rows
  const Tiles tl = tiles_of<kTileN>(a, s, row0 / a.G, (row0 + rows - 1) / a.G + 1);
  const int all_tiles = tl.sink + tl.main;
  const int first = static_cast<int>(static_cast<int64_t>(all_tiles) * blockIdx.z / a.splits);
  const int n_tiles = static_cast<int>(static_cast<int64_t>(all_tiles) * (blockIdx.z + 1) / a.splits) - first;
  auto kv_of = [&](int t) { return tile_at(tl, first + t) * kTileN; };
  // V rows of the tile that no row of this CTA sees
  auto edge = [&](int kv0) { return kv0 + kTileN - 1 > tl.lmax || (kv0 < tl.lmin && kv0 + kTileN - 1 >= a.sinks); };

  uint8_t* sQ = smem;
  auto k_ptr = [&](int st) { return smem + Sh::kK0 + st * Sh::kOperand; };
  auto v_ptr = [&](int st) { return smem + Sh::kV0 + st * Sh::kOperand; };

  if (warp >= 2 && n_tiles > 0) {
    // q rows into the 128-byte-swizzled tiles; rows behind the last are zeros
    for (int x = threadIdx.x - 64; x < n_q * kTileM * (D / 8); x += kTileLoadWarps * 32) {
      const int r = x / (D / 8), ch = x % (D / 8);
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows) {
        const int pr = row0 + r, j = pr / a.G, hq = h * a.G + pr % a.G;
        v = __ldg(reinterpret_cast<const uint4*>(a.q + static_cast<int64_t>(s.q0 + j) * a.q_st +
                                                 static_cast<int64_t>(hq) * a.q_sh) + ch);
      }
      const int rr = r & 127;
      *reinterpret_cast<uint4*>(sQ + (r >> 7) * Sh::kOperand + (ch >> 3) * Sh::kHalfBytes + rr * 128 +
                                (((ch & 7) ^ (rr & 7)) << 4)) = v;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
  }

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    const int page = 1 << a.page_log2;
    const int box = min(page, kTileN);
    const int pieces = kTileN / box;
    const int32_t* row = a.table + static_cast<int64_t>(seq) * a.table_st;
    auto page_of = [&](int t) {
      if (lane >= pieces || t >= n_tiles) return -1;
      const int key = kv_of(t) + lane * box;
      const int p = key >> a.page_log2;
      if (key >= s.kv || p >= a.W) return -1;
      const int id = __ldg(row + p);
      if ((id < 0 || id >= a.pages) && a.status) atomicExch(a.status, QIK_DEV_BAD_INDEX);
      return id < a.pages ? id : -1;
    };
    auto load = [&](const CUtensorMap* tm, uint8_t* dst, int t, int id, uint64_t* bar) {
      if (lane == 0) mbar_arrive_expect_tx(bar, Sh::kOperand);
      __syncwarp();
      if (lane < pieces) {
        const int place = (kv_of(t) + lane * box) & (page - 1);
#pragma unroll
        for (int hd = 0; hd < Sh::kHalves; ++hd)
          tma_load_5d(dst + hd * Sh::kHalfBytes + lane * box * 128, tm, 0, place, hd, h, id, bar);
      }
    };
    // step u: K of tile u, then V of tile u - 1
    int next = page_of(0), cur = -1, prev;
    for (int u = 0; u <= n_tiles && n_tiles > 0; ++u) {
      prev = cur;
      cur = next;
      next = page_of(u + 1);
      if (u < n_tiles) {
        const int st = u & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&k_empty[st], ((u >> 1) & 1) ^ 1u, abort_flag, a.status))) break;
        load(&tm_k, k_ptr(st), u, cur, &k_full[st]);
      }
      const int t = u - 1;
      if (t >= 0) {
        const int st = t & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&v_empty[st], ((t >> 1) & 1) ^ 1u, abort_flag, a.status))) break;
        load(&tm_v, v_ptr(st), t, prev, edge(kv_of(t)) ? &v_raw[st] : &v_full[st]);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && n_tiles > 0) {
      constexpr uint32_t fmt = F16 ? 0 : 1;
      constexpr uint32_t idesc_s = idesc_f32acc(fmt, fmt, 0, 0, kTileM, kTileN);
      constexpr uint32_t idesc_o = idesc_f32acc(fmt, fmt, 0, 1, kTileM, D);
      bool ok = mbar_wait(q_full, 0, abort_flag, a.status);
      tc_fence_after();
      const uint64_t q_desc = sdesc_sw128(smem_u32(sQ), 16, 1024);
      const uint64_t k_desc = sdesc_sw128(smem_u32(k_ptr(0)), 16, 1024);
      const uint64_t v_desc = sdesc_sw128(smem_u32(v_ptr(0)), Sh::kHalfBytes, 1024);
      constexpr uint64_t kOp16 = Sh::kOperand >> 4;
      auto issue_s = [&](int g, int t) {
        const uint64_t qd = q_desc + g * kOp16, kd = k_desc + static_cast<uint64_t>(t & 1) * kOp16;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off16 = ((k >> 2) * Sh::kHalfBytes + (k & 3) * 32) >> 4;
          umma_f16_ss(tmem + 128u * g, qd + off16, kd + off16, idesc_s, k > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[g]);
      };
      auto wait_k = [&](int t) -> bool {
        if (!mbar_wait(&k_full[t & 1], (t >> 1) & 1, abort_flag, a.status)) return false;
        tc_fence_after();
        return true;
      };
      auto issue_pv = [&](int g, int t) -> bool {
        const int st = t & 1;
        if (!mbar_wait(&p_full[g], t & 1, abort_flag, a.status)) return false;
        if (g == 0 && !mbar_wait(&v_full[st], (t >> 1) & 1, abort_flag, a.status)) return false;
        tc_fence_after();
        const uint64_t vd = v_desc + static_cast<uint64_t>(st) * kOp16;
#pragma unroll
        for (int k = 0; k < kTileN / 16; ++k) {
          const uint32_t p_col = 128u * g + k * 8 + (k >= kTileN / 32 ? 32u : 0u);
          umma_f16_ts(tmem + 256u + 128u * g, tmem + p_col, vd + k * 128u, idesc_o, (t > 0 || k > 0) ? 1u : 0u);
        }
        if (t == n_tiles - 1) umma_commit(&o_full[g]);
        if (g == n_q - 1) umma_commit(&v_empty[st]);
        return true;
      };
      if (ok && wait_k(0)) {
        for (int g = 0; g < n_q; ++g) issue_s(g, 0);
        umma_commit(&k_empty[0]);
        for (int t = 0; t < n_tiles && ok; ++t) {
          const bool more = t + 1 < n_tiles;
          for (int g = 0; g < n_q && ok; ++g) {
            ok = issue_pv(g, t);
            if (ok && more) {
              if (g == 0) ok = wait_k(t + 1);
              if (ok) issue_s(g, t + 1);
            }
          }
          if (ok && more) umma_commit(&k_empty[(t + 1) & 1]);
        }
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ V rows nobody sees
    uint32_t seen[2] = {0u, 0u};
    for (int t = 0; t < n_tiles; ++t) {
      const int kv0 = kv_of(t), st = t & 1;
      if (!edge(kv0)) continue;
      if (!__all_sync(0xffffffffu, mbar_wait(&v_raw[st], seen[st]++ & 1u, abort_flag, a.status))) break;
      for (int key = lane >> 3; key < kTileN; key += 4) {
        const int kv = kv0 + key;
        if (kv > tl.lmax || (kv < tl.lmin && kv >= a.sinks)) {
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
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax (tile g)
    const int sw = warp - 4;
    const int g = sw >> 3;
    const int quarter = sw & 3;      // TMEM lane quarter (warp % 4)
    const int sub = (sw >> 2) & 1;   // its lower or upper 16 lanes
    const int hc = lane >> 4;        // column half of the row
    const int r = g * kTileM + quarter * 32 + sub * 16 + (lane & 15);
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32 + sub * 16) << 16;
    const uint32_t tS = tmem + lane_base + 128u * g;
    const uint32_t tO = tmem + lane_base + 256u + 128u * g;
    const int pr = row0 + min(r, rows - 1);  // rows behind the last follow it and are not stored
    const int j = pr / a.G, hq = h * a.G + pr % a.G;
    const int my_last = last_key(a, s, j), my_first = first_key(a, my_last);
    float m_run = -INFINITY, l_run = 0.0f;
    bool ok = true;
    const int work = g < n_q ? n_tiles : 0;
    for (int t = 0; t < work; ++t) {
      if (!__all_sync(0xffffffffu, mbar_wait(&s_full[g], t & 1, abort_flag, a.status))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int kv0 = kv_of(t);
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
          mx[0] = fmax3_nan(mx[0], sv[c], sv[c + 1]);
          mx[1] = fmax3_nan(mx[1], sv[c + 2], sv[c + 3]);
          mx[2] = fmax3_nan(mx[2], sv[c + 4], sv[c + 5]);
          mx[3] = fmax3_nan(mx[3], sv[c + 6], sv[c + 7]);
        }
      } else {
        const int col0 = kv0 + 64 * hc;
        const int last = my_last - col0, low = my_first - col0, sink = a.sinks - col0;
#pragma unroll
        for (int c = 0; c < 64; ++c) {
          sv[c] = c <= last && (c >= low || c < sink) ? sv[c] : -INFINITY;
          mx[c & 3] = fmaxf(mx[c & 3], sv[c]);
        }
      }
      // a NaN score reaches the row's sum through its maximum: 2^x on the FMA pipe clamps it
      float raw_max = fmax3_nan(mx[0], mx[1], mx[2]);
      raw_max = fmax3_nan(raw_max, mx[3], __shfl_xor_sync(0xffffffffu, fmax3_nan(raw_max, mx[3], mx[3]), 16));
      const float tmax = raw_max * a.scale_log2;
      float alpha = 1.0f;
      bool rescale = false;
      if (tmax > m_run + kTileRescale || (m_run == -INFINITY && tmax > -INFINITY)) {
        rescale = m_run != -INFINITY;
        alpha = rescale ? ex2(m_run - tmax) : 0.0f;
        m_run = tmax;
      }
      const float neg_m = m_run == -INFINITY ? 0.0f : -m_run;
      const float psum = whole ? tile_softmax<true, F16>(sv, a.scale_log2, neg_m, tS)
                               : tile_softmax<false, F16>(sv, a.scale_log2, neg_m, tS);
      l_run = l_run * alpha + (raw_max == raw_max ? psum : raw_max);
      if (t >= 1 && __any_sync(0xffffffffu, rescale)) {
        const float f = rescale ? alpha : 1.0f;
        uint32_t rr[kHalfO];
        tmem_ld_half<D>(tO, rr);
#pragma unroll
        for (int i = 0; i < kHalfO; ++i) rr[i] = __float_as_uint(__uint_as_float(rr[i]) * f);
        tmem_st_half<D>(tO, rr);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[g]);
    }
    // ---- O / l, or the piece of this split
    const float l_row = l_run + __shfl_xor_sync(0xffffffffu, l_run, 16);
    float o[kHalfO];
#pragma unroll
    for (int i = 0; i < kHalfO; ++i) o[i] = 0.0f;
    const bool ready = ok && work > 0 && mbar_wait(&o_full[g], 0, abort_flag, a.status);
    if (__all_sync(0xffffffffu, ready)) {
      tc_fence_after();
      uint32_t rr[kHalfO];
      tmem_ld_half<D>(tO, rr);
#pragma unroll
      for (int i = 0; i < kHalfO; ++i) o[i] = __uint_as_float(rr[i]);
    }
    if (r < rows && a.splits == 1) {
      const float inv = l_row == 0.0f ? 0.0f : 1.0f / l_row;
      uint16_t* dst = a.out + static_cast<int64_t>(s.q0 + j) * a.o_st + static_cast<int64_t>(hq) * a.o_sh + kHalfO * hc;
#pragma unroll
      for (int c = 0; c < kHalfO; c += 8)
        *reinterpret_cast<uint4*>(dst + c) =
            make_uint4(pack16<F16>(o[c] * inv, o[c + 1] * inv), pack16<F16>(o[c + 2] * inv, o[c + 3] * inv),
                       pack16<F16>(o[c + 4] * inv, o[c + 5] * inv), pack16<F16>(o[c + 6] * inv, o[c + 7] * inv));
    } else if (r < rows) {
      const int64_t at = ((static_cast<int64_t>(blockIdx.z) * gridDim.y + block) * a.HK + h) * kTileRows + r;
      float* dst = a.ws_o + at * D + kHalfO * hc;
#pragma unroll
      for (int c = 0; c < kHalfO; c += 4)
        *reinterpret_cast<float4*>(dst + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
      if (hc == 0) a.ws_ml[at] = make_float2(m_run, l_row);
    }
  }
  tc_fence_before();
  __syncthreads();
  pdl_trigger();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the splits of a 256-row block in split order.  One warp a row.
template <int D, bool F16>
__global__ void __launch_bounds__(256) paged_tile_join_kernel(const PagedDev a) {
  __shared__ int slot[2 + 8];
  pdl_wait();
  const int block = blockIdx.y, h = blockIdx.x;
  if (!find_block(a, block, slot, 8)) return;
  const Seq s = seq_of(a, slot[0]);
  const int row0 = slot[1] * kTileRows, rows = min(s.n * a.G - row0, kTileRows);
  const int64_t pitch = static_cast<int64_t>(gridDim.y) * a.HK * kTileRows;
  for (int r = blockIdx.z * 8 + (threadIdx.x >> 5); r < rows; r += 8 * gridDim.z) {
    const int64_t at = (static_cast<int64_t>(block) * a.HK + h) * kTileRows + r;
    const int pr = row0 + r;
    join_row<D, F16>(a, a.splits, [&](int z) { return at + z * pitch; },
                     a.out + static_cast<int64_t>(s.q0 + pr / a.G) * a.o_st + static_cast<int64_t>(h * a.G + pr % a.G) * a.o_sh);
  }
  pdl_trigger();
}

// ============================================================ host
constexpr int kSplitRows = 64;  // most rows of a sequence that the split kernel takes

struct PagedPlan {
  bool split, tile, unit_mode;
  int split_mt, split_ctas, tile_blocks, tile_splits;
  size_t split_o, split_ml, split_desc, tile_o, tile_ml, bytes;  // workspace offsets
};

static PagedPlan paged_plan(const qik_paged_attn_args& A) {
  PagedPlan p = {};
  const int64_t G = A.HQ / A.HK, max_rows = A.max_new * G;
  const int sms = sm_count();
  // sequences of at most kSplitRows rows may exist unless all have max_new tokens
  p.tile = max_rows > kSplitRows;
  p.split = !p.tile || A.T != A.B * A.max_new;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  if (p.split) {
    p.split_mt = max_rows <= 16 ? 1 : max_rows <= 32 ? 2 : 4;
    // short contexts (at most 8 tiles): one CTA for each (sequence, head), nothing to join
    p.unit_mode = A.max_kv <= 8 * kSplitTile;
    p.split_ctas = p.unit_mode ? static_cast<int>(A.B * A.HK) : sms * (p.split_mt == 1 ? 2 : 1);
    if (!p.unit_mode) {
      const size_t rows = static_cast<size_t>(2) * p.split_ctas * p.split_mt * 16;
      p.split_o = take(rows * A.D * sizeof(float));
      p.split_ml = take(rows * sizeof(float2));
      p.split_desc = take(p.split_ctas * sizeof(int4));
    }
  }
  if (p.tile) {
    const int64_t by_rows = A.T * G / kTileRows + A.B, by_seq = A.B * ((max_rows + kTileRows - 1) / kTileRows);
    p.tile_blocks = static_cast<int>(by_rows < by_seq ? by_rows : by_seq);
    // few blocks: the keys are split over CTAs until the GPU is full, at least 4 tiles each
    const int64_t ctas = static_cast<int64_t>(p.tile_blocks) * A.HK, tiles = (A.max_kv + kTileN - 1) / kTileN;
    int64_t splits = ctas >= sms ? 1 : sms / ctas;
    if (splits > tiles / 4) splits = tiles / 4;
    p.tile_splits = splits < 1 ? 1 : static_cast<int>(splits);
    if (p.tile_splits > 1) {
      const size_t rows = static_cast<size_t>(p.tile_splits) * ctas * kTileRows;
      p.tile_o = take(rows * A.D * sizeof(float));
      p.tile_ml = take(rows * sizeof(float2));
    }
  }
  p.bytes = at;
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
  QIK_REQUIRE(A.W >= 0 && A.W * A.page <= (1ll << 30), "qik_paged_attention: page table of %lld columns", (long long)A.W);
  QIK_REQUIRE(A.B * A.HK <= 0x7FFFFFFFll && A.B * A.HK * (A.W * A.page / kSplitTile + 3) <= 0x7FFFFFFFll,
              "qik_paged_attention: %lld sequences of up to %lld keys are too much for one call", (long long)A.B,
              (long long)(A.W * A.page));
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
  e = launch_kernel(paged_split_kernel<D, MT, TEAMS, F16>, dim3(ctas), dim3(Sh::kThreads), Sh::kBytes, st, true, tk, tv, d);
  if (e != cudaSuccess || d.unit_mode) return e;
  return launch_kernel(paged_split_join_kernel<D, F16>, dim3(ctas, MT * 4), dim3(128), 0, st, true, d, MT * 16);
}
template <int D, bool F16>
static cudaError_t launch_paged(const qik_paged_attn_args& A, const PagedPlan& p, PagedDev d, uint8_t* ws,
                                const CUtensorMap* maps, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  if (p.split) {
    PagedDev s = d;
    s.lo_rows = 0;
    s.hi_rows = p.split_mt * 16;
    s.unit_mode = p.unit_mode;
    s.ws_o = reinterpret_cast<float*>(ws + p.split_o);
    s.ws_ml = reinterpret_cast<float2*>(ws + p.split_ml);
    s.ws_desc = reinterpret_cast<int4*>(ws + p.split_desc);
    const bool few = p.unit_mode && p.split_ctas <= sm_count();
    e = p.split_mt == 1   ? (few ? launch_split<D, 1, 2, F16>(maps[0], maps[1], s, p.split_ctas, st)
                                 : launch_split<D, 1, 1, F16>(maps[0], maps[1], s, p.split_ctas, st))
        : p.split_mt == 2 ? launch_split<D, 2, 1, F16>(maps[0], maps[1], s, p.split_ctas, st)
                          : launch_split<D, 4, 1, F16>(maps[0], maps[1], s, p.split_ctas, st);
    if (e != cudaSuccess) return e;
  }
  if (p.tile) {
    using Sh = TileShape<D>;
    static std::once_flag once[64];
    e = allow_smem(paged_tile_kernel<D, F16>, Sh::kBytes, once);
    if (e != cudaSuccess) return e;
    d.lo_rows = kSplitRows;
    d.hi_rows = 0x7FFFFFFF;
    d.splits = p.tile_splits;
    d.ws_o = reinterpret_cast<float*>(ws + p.tile_o);
    d.ws_ml = reinterpret_cast<float2*>(ws + p.tile_ml);
    const dim3 grid(static_cast<unsigned>(A.HK), static_cast<unsigned>(p.tile_blocks), static_cast<unsigned>(p.tile_splits));
    e = launch_kernel(paged_tile_kernel<D, F16>, grid, dim3(kTileThreads), Sh::kBytes, st, true, maps[2], maps[3], d);
    if (e != cudaSuccess || p.tile_splits == 1) return e;
    const dim3 jgrid(static_cast<unsigned>(A.HK), static_cast<unsigned>(p.tile_blocks), 8);
    e = launch_kernel(paged_tile_join_kernel<D, F16>, jgrid, dim3(256), 0, st, true, d);
  }
  return e;
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
                  A.kp_s0 >= 0 && A.kp_sh >= 0 && A.kp_ss > 0 && A.vp_s0 >= 0 && A.vp_sh >= 0 && A.vp_ss > 0,
              "qik_paged_attention: strides must be multiples of 8 elements");
  const PagedPlan p = paged_plan(A);
  QIK_REQUIRE(p.bytes == 0 || (ws && ws_bytes >= p.bytes), "qik_paged_attention: workspace of %zu bytes, %zu needed",
              ws_bytes, p.bytes);
  QIK_REQUIRE(p.tile_blocks <= 65535, "qik_paged_attention: %d row blocks are too many (65535)", p.tile_blocks);
  const bool f16 = (A.flags & QIK_PAGED_F16) != 0;
  CUtensorMap maps[4];
  if (p.split) {
    rc = page_map(&maps[0], A.k_pages, f16, A, A.kp_s0, A.kp_sh, A.kp_ss, kSplitTile, static_cast<uint32_t>(A.D / 64));
    if (!rc) rc = page_map(&maps[1], A.v_pages, f16, A, A.vp_s0, A.vp_sh, A.vp_ss, kSplitTile, static_cast<uint32_t>(A.D / 64));
  }
  if (!rc && p.tile) {
    rc = page_map(&maps[2], A.k_pages, f16, A, A.kp_s0, A.kp_sh, A.kp_ss, kTileN, 1);
    if (!rc) rc = page_map(&maps[3], A.v_pages, f16, A, A.vp_s0, A.vp_sh, A.vp_ss, kTileN, 1);
  }
  if (rc) return rc;
  PagedDev d = {};
  d.q = static_cast<const uint16_t*>(A.q);
  d.out = static_cast<uint16_t*>(A.out);
  d.table = A.page_table, d.lens = A.seq_lens, d.starts = A.query_starts;
  d.status = status;
  d.q_st = A.q_st, d.q_sh = A.q_sh, d.o_st = A.o_st, d.o_sh = A.o_sh, d.table_st = A.table_st;
  d.B = static_cast<int>(A.B), d.T = static_cast<int>(A.T), d.HK = static_cast<int>(A.HK);
  d.G = static_cast<int>(A.HQ / A.HK), d.W = static_cast<int>(A.W), d.pages = static_cast<int>(A.pages);
  while ((1ll << d.page_log2) < A.page) ++d.page_log2;
  d.max_new = static_cast<int>(A.max_new);
  d.window = A.window, d.sinks = A.window > 0 ? A.sinks : 0;
  d.splits = 1, d.min_share = 4;
  d.scale_log2 = A.sm_scale * 1.4426950408889634f;
  d.causal = (A.flags & QIK_PAGED_CAUSAL) != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* w = static_cast<uint8_t*>(ws);
  cudaError_t e = A.D == 128 ? (f16 ? launch_paged<128, true>(A, p, d, w, maps, st) : launch_paged<128, false>(A, p, d, w, maps, st))
                             : (f16 ? launch_paged<64, true>(A, p, d, w, maps, st) : launch_paged<64, false>(A, p, d, w, maps, st));
  QIK_TRY_CUDA(e);
  return check_launch("qik_paged_attention");
}
