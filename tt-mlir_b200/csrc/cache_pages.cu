// Upkeep of paged key / value caches [blocks, heads, block_size, head_dim], for all caches of a model in one launch:
//  ttb_paged_copy_blocks   whole blocks dst <- src: a sequence forks (its last, partly filled block is duplicated),
//                          beams are reordered, live blocks move into holes before the pool shrinks
//  ttb_paged_commit_draft  the accepted path of a verified draft tree is appended to its user's cached sequence
// Both only move bytes: the bound is HBM (each byte read and written once), or the launch when there is little to move.
// Measured: 96 blocks of 64 KB in 32 caches 55.6 us (6.3 TB/s: the 96 have some 72 sources), one block in 2 caches 8.6 (1.6 of
// it on the GPU); the paths of 48 users (up to 31 rows of 2 KB) in 32 caches 20.2 us (4.8 TB/s; 29.6 with the places looked
// up per cache).
#include "common.cuh"

#include <algorithm>

namespace ttb {

constexpr int PG_CACHES = 256;  // cache pointers per launch (kernel parameters); more caches take more launches
constexpr int PG_THREADS = 256;
constexpr int PG_UNROLL = 4;    // units in flight per thread
constexpr int PG_PAIRS = 1 << 20; // pairs per call: every one is checked against the whole list

struct PagePointers {
  void *cache[PG_CACHES];
};
struct DraftPointers {
  void *cache[PG_CACHES];
  const void *draft[PG_CACHES];
};

// grid: x = pair * pieces + piece of the block, y = group of caches.  A pair is executed only when no other pair reads
// its destination and no earlier pair writes it, so that the result does not depend on the order in which CTAs run;
// every CTA checks that for its own pair against the whole list while its first loads are in flight.  With a long list a CTA
// moves its piece in several caches, so that it reads no more of the list than it moves.
template <typename U>
__global__ void __launch_bounds__(PG_THREADS)
    copyBlocksKernel(PagePointers ptrs, int caches, const int2 *__restrict__ pairs, int n, int64_t blocks, int64_t blockUnits, int pieces, int *bad) {
  pdlLaunchDependents();
  pdlWait();
  const int pair = blockIdx.x / pieces, piece = blockIdx.x % pieces;
  const int2 pr = pairs[pair];
  if (pr.x < 0 && pr.y < 0) return; // padding
  if (pr.x < 0 || pr.y < 0 || pr.x >= blocks || pr.y >= blocks) {
    if (threadIdx.x == 0) *bad = 1;
    return;
  }
  if (pr.x == pr.y) return;
  const int64_t from = static_cast<int64_t>(piece) * (PG_THREADS * PG_UNROLL) + threadIdx.x;
  U r[PG_UNROLL];
  auto load = [&](const U *src) {
#pragma unroll
    for (int i = 0; i < PG_UNROLL; ++i) {
      if (from + i * PG_THREADS < blockUnits) r[i] = src[from + i * PG_THREADS];
    }
  };
  auto store = [&](U *dst) {
#pragma unroll
    for (int i = 0; i < PG_UNROLL; ++i) {
      if (from + i * PG_THREADS < blockUnits) dst[from + i * PG_THREADS] = r[i];
    }
  };
  int c = blockIdx.y;
  load(static_cast<const U *>(ptrs.cache[c]) + pr.x * blockUnits);
  int clash = 0;
  for (int i = threadIdx.x; i < n; i += PG_THREADS) {
    const int2 o = pairs[i];
    if (i != pair && (o.x == pr.y || (o.y == pr.y && i < pair))) clash = 1;
  }
  if (__syncthreads_or(clash)) {
    if (threadIdx.x == 0) *bad = 1;
    return;
  }
  for (;;) {
    store(static_cast<U *>(ptrs.cache[c]) + pr.y * blockUnits);
    c += gridDim.y;
    if (c >= caches) return;
    load(static_cast<const U *>(ptrs.cache[c]) + pr.x * blockUnits);
  }
}

// grid: x = piece of a user's [nodes, heads, row] items, y = user, z = group of caches.  Item i of the path goes to
// position lens[b] + i.  Where a unit comes from and goes to is the same in every cache and costs a chain of dependent
// loads (length, path, page), so a CTA finds it once and then moves its units in one cache after the other, the next
// cache's loads in front of this one's stores.
template <typename U>
__global__ void __launch_bounds__(PG_THREADS)
    commitDraftKernel(DraftPointers ptrs, int caches, const int32_t *__restrict__ table, const int32_t *__restrict__ lens, const int32_t *__restrict__ path,
                      const int32_t *__restrict__ pathLens, int nodes, int heads, int64_t blocks, int blockSize, int pages, int rowUnits, int *bad) {
  pdlLaunchDependents();
  pdlWait();
  const int b = blockIdx.y, perNode = heads * rowUnits;
  const int count = min(max(pathLens[b], 0), nodes);
  const int64_t total = static_cast<int64_t>(count) * perNode;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (PG_THREADS * PG_UNROLL);
  if (first >= total) return;
  const int64_t len = lens[b];
  int64_t src[PG_UNROLL], dst[PG_UNROLL];
#pragma unroll
  for (int i = 0; i < PG_UNROLL; ++i) {
    const int64_t at = first + i * PG_THREADS + threadIdx.x;
    dst[i] = -1;
    if (at >= total) continue;
    const bool small = total <= 0x7fffffff; // a 64-bit division costs several times a 32-bit one
    const int step = small ? static_cast<int>(at) / perNode : static_cast<int>(at / perNode);
    const int rem = static_cast<int>(at - static_cast<int64_t>(step) * perNode), h = rem / rowUnits, u = rem % rowUnits;
    const int node = path[static_cast<int64_t>(b) * nodes + step];
    const int64_t pos = len + step;
    const int64_t page = pos <= 0x7fffffff ? static_cast<int>(pos) / blockSize : pos / blockSize;
    int blk = -1;
    if (len >= 0 && page < pages) blk = table[static_cast<int64_t>(b) * pages + page];
    if (node < 0 || node >= nodes || blk < 0 || blk >= blocks) { // nowhere to go: left out and reported
      *bad = 1;
      continue;
    }
    src[i] = (static_cast<int64_t>(b) * nodes + node) * perNode + rem;
    dst[i] = ((blk * static_cast<int64_t>(heads) + h) * blockSize + (pos - page * blockSize)) * rowUnits + u;
  }
  U r[PG_UNROLL], next[PG_UNROLL];
  auto load = [&](U *to, const void *draft) {
#pragma unroll
    for (int i = 0; i < PG_UNROLL; ++i) {
      if (dst[i] >= 0) to[i] = static_cast<const U *>(draft)[src[i]];
    }
  };
  int c = blockIdx.z;
  load(r, ptrs.draft[c]);
  for (;;) {
    const int after = c + gridDim.z;
    if (after < caches) load(next, ptrs.draft[after]);
    U *cache = static_cast<U *>(ptrs.cache[c]);
#pragma unroll
    for (int i = 0; i < PG_UNROLL; ++i) {
      if (dst[i] >= 0) cache[dst[i]] = r[i];
      r[i] = next[i];
    }
    if (after >= caches) return;
    c = after;
  }
}

// Largest power of two up to 16 that divides `bytes` and every pointer.
static int unitOf(int64_t bytes, void *const *a, const void *const *b, int n) {
  uintptr_t bits = static_cast<uintptr_t>(bytes) | 16;
  for (int i = 0; i < n; ++i) {
    bits |= reinterpret_cast<uintptr_t>(a[i]);
    if (b) bits |= reinterpret_cast<uintptr_t>(b[i]);
  }
  return static_cast<int>(bits & (~bits + 1));
}

#define TTB_PAGE_UNITS(unit, U, ...)                                     \
  switch (unit) {                                                        \
  case 16: { using U = uint4; __VA_ARGS__; } break;                      \
  case 8: { using U = uint2; __VA_ARGS__; } break;                       \
  case 4: { using U = uint32_t; __VA_ARGS__; } break;                    \
  case 2: { using U = uint16_t; __VA_ARGS__; } break;                    \
  default: { using U = uint8_t; __VA_ARGS__; } break;                    \
  }

int indexBadFlag(int **flag); // index_ops.cu: the word that ttb_index_status reports

} // namespace ttb

using namespace ttb;

extern "C" {

int ttb_paged_copy_blocks(void *const *host_caches, int n_caches, const void *pairs, int n_pairs, int dtype, int64_t blocks, int64_t heads,
                          int64_t block_size, int64_t head_dim, void *stream) {
  TTB_CHECK(n_caches >= 0 && n_pairs >= 0, "negative count");
  TTB_CHECK(n_pairs <= PG_PAIRS, "a call takes at most 2^20 pairs");
  TTB_CHECK(blocks > 0 && heads > 0 && block_size > 0 && head_dim > 0, "empty paged cache");
  TTB_CHECK(blocks <= 0x7fffffff && heads <= 1 << 24 && block_size <= 1 << 24 && head_dim <= 1 << 24, "cache extents are too large");
  const int64_t es = static_cast<int64_t>(dtypeSize(dtype));
  TTB_CHECK(es > 0, "unsupported dtype");
  if (n_caches == 0 || n_pairs == 0) return TTB_OK;
  TTB_CHECK(host_caches && pairs, "null tensor");
  TTB_CHECK((reinterpret_cast<uintptr_t>(pairs) & 7) == 0, "pairs must be 8-byte aligned");
  const double bytes = double(heads) * double(block_size) * double(head_dim) * double(es);
  TTB_CHECK(bytes <= double(int64_t(1) << 40), "a block is limited to 2^40 bytes");
  for (int i = 0; i < n_caches; ++i) TTB_CHECK(host_caches[i], "null cache");
  const int64_t blockBytes = heads * block_size * head_dim * es;
  const int unit = unitOf(blockBytes, host_caches, nullptr, n_caches);
  const int64_t units = blockBytes / unit, pieces = (units + PG_THREADS * PG_UNROLL - 1) / (PG_THREADS * PG_UNROLL);
  TTB_CHECK(pieces * n_pairs <= 0x7fffffff, "too much to move in one call");
  int *bad = nullptr;
  const int rc = indexBadFlag(&bad);
  if (rc) return rc;
  cudaStream_t st = asStream(stream);
  ProfScope prof("paged_copy_blocks", 0, 2.0 * bytes * n_pairs * n_caches, st);
  for (int c0 = 0; c0 < n_caches; c0 += PG_CACHES) {
    PagePointers ptrs;
    const int n = std::min(PG_CACHES, n_caches - c0);
    for (int i = 0; i < n; ++i) ptrs.cache[i] = host_caches[c0 + i];
    // Measured, a CTA per cache / all caches by one CTA, us: 10000 pairs of 2 KB in 8 caches 510 / 131, 4096 pairs of 64 KB in
    // 32 caches 2584 / 2710, 96 of them 55.5 / 57.
    const int64_t moved = 2 * std::min<int64_t>(blockBytes, int64_t(PG_THREADS) * PG_UNROLL * unit), read = int64_t(sizeof(int2)) * n_pairs;
    const int64_t each = (read + moved - 1) / moved, groups = (n + each - 1) / each;
    dim3 grid(static_cast<unsigned>(pieces * n_pairs), static_cast<unsigned>(groups));
    TTB_PAGE_UNITS(unit, U, TTB_CUDA(launchPdl(copyBlocksKernel<U>, grid, dim3(PG_THREADS), 0, st, ptrs, n, static_cast<const int2 *>(pairs), n_pairs,
                                               blocks, units, static_cast<int>(pieces), bad)))
    countLaunch();
  }
  TTB_LAUNCH_CHECK();
  return TTB_OK;
}

int ttb_paged_commit_draft(void *const *host_caches, const void *const *host_drafts, int n_caches, const void *page_table,
                           const void *cached_lens, const void *path, const void *path_lens, int dtype, int64_t users, int64_t nodes,
                           int64_t heads, int64_t blocks, int64_t block_size, int64_t pages, int64_t head_dim, void *stream) {
  TTB_CHECK(n_caches >= 0 && users >= 0 && nodes >= 0, "negative count");
  TTB_CHECK(blocks > 0 && heads > 0 && block_size > 0 && pages > 0 && head_dim > 0, "empty paged cache");
  TTB_CHECK(users <= 65535, "users are limited to 65535");
  TTB_CHECK(blocks <= 0x7fffffff && block_size <= 1 << 24 && pages <= 1 << 24 && heads <= 1 << 24 && head_dim <= 1 << 24 && nodes <= 1 << 24,
            "cache extents are too large");
  const int64_t es = static_cast<int64_t>(dtypeSize(dtype));
  TTB_CHECK(es > 0, "unsupported dtype");
  TTB_CHECK(heads * head_dim * es <= 0x7fffffff, "a token's row is limited to 2^31 bytes");
  if (n_caches == 0 || users == 0 || nodes == 0) return TTB_OK;
  TTB_CHECK(host_caches && host_drafts && page_table && cached_lens && path && path_lens, "null tensor");
  TTB_CHECK(alignedTo(4, page_table, cached_lens, path, path_lens), "tensors must be aligned to their elements");
  for (int i = 0; i < n_caches; ++i) TTB_CHECK(host_caches[i] && host_drafts[i], "null cache or draft");
  const int unit = unitOf(head_dim * es, host_caches, host_drafts, n_caches);
  const int rowUnits = static_cast<int>(head_dim * es / unit);
  const int64_t pieces = (nodes * heads * rowUnits + PG_THREADS * PG_UNROLL - 1) / (PG_THREADS * PG_UNROLL);
  TTB_CHECK(pieces <= 0x7fffffff, "too much to move in one call");
  int *bad = nullptr;
  const int rc = indexBadFlag(&bad);
  if (rc) return rc;
  cudaStream_t st = asStream(stream);
  ProfScope prof("paged_commit_draft", 0, 2.0 * n_caches * users * nodes * heads * head_dim * es, st); // an upper bound
  for (int c0 = 0; c0 < n_caches; c0 += PG_CACHES) {
    DraftPointers ptrs;
    const int n = std::min(PG_CACHES, n_caches - c0);
    for (int i = 0; i < n; ++i) {
      ptrs.cache[i] = host_caches[c0 + i];
      ptrs.draft[i] = host_drafts[c0 + i];
    }
    // as many groups of caches as fill the GPU twice over (paths are often half as long as they may be)
    const int64_t fill = 2 * smCount() * (2048 / PG_THREADS);
    const int64_t groups = std::min<int64_t>(n, std::max<int64_t>(1, fill / (pieces * users)));
    dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(users), static_cast<unsigned>(groups));
    TTB_PAGE_UNITS(unit, U, TTB_CUDA(launchPdl(commitDraftKernel<U>, grid, dim3(PG_THREADS), 0, st, ptrs, n, static_cast<const int32_t *>(page_table),
                                               static_cast<const int32_t *>(cached_lens), static_cast<const int32_t *>(path),
                                               static_cast<const int32_t *>(path_lens), static_cast<int>(nodes), static_cast<int>(heads), blocks,
                                               static_cast<int>(block_size), static_cast<int>(pages), rowUnits, bad)))
    countLaunch();
  }
  TTB_LAUNCH_CHECK();
  return TTB_OK;
}

} // extern "C"
