// qik_pages.cu -- copies between pages of a paged KV cache: what a fork (the child's own
// copy of a partly filled page) and a compaction (pages moved down into holes) need on
// the device.
//
// The lists come from the host, which owns the allocation: they are checked there
// (every index in range, destinations distinct and never also read in the call) and
// travel as kernel parameters, so there is no copy to the device to wait for and no
// list whose lifetime the caller has to keep.
//
// Bound by HBM (read + write of the moved tokens).  A page holds [head][token][D], so
// the first t tokens of each head are one run of t * D elements.
#include <new>

#include "qik_device.cuh"
#include "qik_host.h"

namespace qik {

constexpr int kPageThreads = 32;
constexpr int kPageUnroll = 16;

template <int N>
struct PageMoves {
  int32_t n;
  int32_t src[N], dst[N], tokens[N];
};

struct PagePools {
  uint8_t* pool[2];            // k pages, v pages
  int64_t layer_bytes[2], page_bytes[2], head_bytes[2];
  int token_bytes, heads, layers, page;
};

// blockIdx.x: (pool, layer, head); blockIdx.y: move; blockIdx.z: 8 KB of the run.  Sixteen loads in flight a
// thread and many small CTAs: 500 whole pages (3.1 GB moved) 506 us with 32 threads x 16, 513 with
// 64 x 16, 535 with 128 x 8, 579 with 128 x 4; bulk copies through shared memory 547 (and 22.5
// instead of 6.8 us for seven partly filled pages).
template <int N>
__global__ void __launch_bounds__(kPageThreads) copy_pages_kernel(const __grid_constant__ PageMoves<N> m,
                                                                  const PagePools p) {
  pdl_wait();
  const int mv = blockIdx.y;
  int u = blockIdx.x;
  const int head = u % p.heads;
  u /= p.heads;
  const int layer = u % p.layers;
  const int which = u / p.layers;
  uint8_t* base = p.pool[which] + layer * p.layer_bytes[which] + head * p.head_bytes[which];
  const uint4* s = reinterpret_cast<const uint4*>(base + m.src[mv] * p.page_bytes[which]);
  uint4* d = reinterpret_cast<uint4*>(base + m.dst[mv] * p.page_bytes[which]);
  const int n = m.tokens[mv] * (p.token_bytes >> 4);
  for (int i0 = blockIdx.z * (kPageThreads * kPageUnroll) + threadIdx.x; i0 < n;
       i0 += gridDim.z * (kPageThreads * kPageUnroll)) {
    uint4 v[kPageUnroll];
#pragma unroll
    for (int j = 0; j < kPageUnroll; ++j)
      if (i0 + j * kPageThreads < n) v[j] = __ldcs(s + i0 + j * kPageThreads);
#pragma unroll
    for (int j = 0; j < kPageUnroll; ++j)
      if (i0 + j * kPageThreads < n) __stcs(d + i0 + j * kPageThreads, v[j]);
  }
  pdl_trigger();
}

template <int N>
static int launch_copy(const int32_t* moves, int64_t n, const PagePools& p, int z, cudaStream_t st) {
  PageMoves<N> m;
  m.n = static_cast<int32_t>(n);
  for (int64_t i = 0; i < n; ++i) m.src[i] = moves[3 * i], m.dst[i] = moves[3 * i + 1], m.tokens[i] = moves[3 * i + 2];
  const dim3 grid(static_cast<unsigned>(2 * p.layers * p.heads), static_cast<unsigned>(n), static_cast<unsigned>(z));
  QIK_TRY_CUDA(launch_kernel(copy_pages_kernel<N>, grid, dim3(kPageThreads), 0, st, true, m, p));
  return check_launch("copy_pages_kernel");
}

}  // namespace qik

using namespace qik;

extern "C" int qik_copy_pages(const qik_page_pools* pools, const int32_t* moves, int64_t n, void* stream) {
  QIK_REQUIRE(pools != nullptr, "qik_copy_pages: pools is NULL");
  const qik_page_pools& A = *pools;
  QIK_REQUIRE(n >= 0 && n <= (1ll << 30), "qik_copy_pages: %lld moves", (long long)n);
  QIK_REQUIRE(A.layers > 0 && A.pages > 0 && A.heads > 0 && A.page > 0 && A.token_bytes > 0 &&
                  A.pages <= 0x7FFFFFFFll && A.layers <= 65535 && A.heads <= 65535 && A.page <= 65536 &&
                  A.token_bytes <= 65536 && 2 * A.layers * A.heads <= 0x7FFFFFFFll,
              "qik_copy_pages: bad sizes (%lld layers, %lld pages, %lld heads, %lld tokens of %lld bytes)",
              (long long)A.layers, (long long)A.pages, (long long)A.heads, (long long)A.page, (long long)A.token_bytes);
  QIK_REQUIRE(A.token_bytes % 16 == 0, "qik_copy_pages: a head's token must be a multiple of 16 bytes, got %lld",
              (long long)A.token_bytes);
  if (n == 0) return QIK_OK;
  QIK_REQUIRE(moves && A.k && A.v, "qik_copy_pages: NULL pointer");
  QIK_REQUIRE(aligned16(A.k) && aligned16(A.v), "qik_copy_pages: pools must be 16-byte aligned");
  QIK_REQUIRE((A.k_layer_bytes | A.k_page_bytes | A.k_head_bytes | A.v_layer_bytes | A.v_page_bytes | A.v_head_bytes) %
                      16 ==
                  0,
              "qik_copy_pages: pool strides must be multiples of 16 bytes");
  // every index in range; no page written twice, none both written and read
  const size_t words = static_cast<size_t>((A.pages + 31) / 32);
  uint32_t* seen = new (std::nothrow) uint32_t[2 * words]();
  if (!seen) return set_error(QIK_ERR_INVALID, "qik_copy_pages: no host memory to check %lld pages", (long long)A.pages);
  uint32_t *read = seen, *written = seen + words;
  int rc = QIK_OK;
  int64_t most = 0;
  for (int64_t i = 0; i < n && rc == QIK_OK; ++i) {
    const int64_t s = moves[3 * i], d = moves[3 * i + 1], t = moves[3 * i + 2];
    if (s < 0 || s >= A.pages || d < 0 || d >= A.pages || t < 0 || t > A.page) {
      rc = set_error(QIK_ERR_INVALID, "qik_copy_pages: move %lld (page %lld to %lld, %lld tokens) is outside %lld pages of %lld tokens",
                     (long long)i, (long long)s, (long long)d, (long long)t, (long long)A.pages, (long long)A.page);
    } else if (written[d >> 5] >> (d & 31) & 1u) {
      rc = set_error(QIK_ERR_INVALID, "qik_copy_pages: page %lld is written twice", (long long)d);
    } else {
      read[s >> 5] |= 1u << (s & 31);
      written[d >> 5] |= 1u << (d & 31);
      most = t > most ? t : most;
    }
  }
  for (size_t w = 0; w < words && rc == QIK_OK; ++w)
    if (read[w] & written[w])
      rc = set_error(QIK_ERR_INVALID, "qik_copy_pages: a page near %lld is both read and written", (long long)w * 32);
  delete[] seen;
  if (rc != QIK_OK) return rc;
  if (most == 0) return QIK_OK;
  PagePools p;
  p.pool[0] = static_cast<uint8_t*>(A.k), p.pool[1] = static_cast<uint8_t*>(A.v);
  p.layer_bytes[0] = A.k_layer_bytes, p.layer_bytes[1] = A.v_layer_bytes;
  p.page_bytes[0] = A.k_page_bytes, p.page_bytes[1] = A.v_page_bytes;
  p.head_bytes[0] = A.k_head_bytes, p.head_bytes[1] = A.v_head_bytes;
  p.token_bytes = static_cast<int>(A.token_bytes), p.heads = static_cast<int>(A.heads);
  p.layers = static_cast<int>(A.layers), p.page = static_cast<int>(A.page);
  // one CTA of one warp for each 8 KB of a head's run (16 vectors a thread)
  const int64_t chunk = kPageThreads * kPageUnroll * 16;
  const int64_t chunks = (most * A.token_bytes + chunk - 1) / chunk;
  const int z = static_cast<int>(chunks < 65535 ? chunks : 65535);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int64_t i = 0; i < n;) {
    const int64_t m = n - i < 320 ? n - i : 320;
    rc = m > 32 ? launch_copy<320>(moves + 3 * i, m, p, z, st) : launch_copy<32>(moves + 3 * i, m, p, z, st);
    if (rc != QIK_OK) return rc;
    i += m;
  }
  return QIK_OK;
}
