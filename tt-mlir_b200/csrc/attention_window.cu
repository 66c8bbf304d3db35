// Attention of a few query rows over a long (usually paged) key / value cache, and attention inside a sliding
// window.  Three entry points share the kernels below:
//  ttb_sdpa_window         a prompt or a chunk of one: row r is the token at position p = r + offset
//  ttb_sdpa_window_decode  one new token per user at position p = cur_pos[b], whose key is already cached
//  ttb_sdpa_tree           a tree of drafted tokens per user behind lens[b] cached ones: node t has position
//                          p = lens[b] + depth(t); its own and its ancestors' keys come from the draft tensors
// out = softmax(scale q k^T) v over the keys that a row sees: key j is seen when j <= p and (j < sinks or
// j > p - window); of the drafted keys a node sees its own and its ancestors', inside the same window.  Scores,
// maxima, sums and the output accumulate in f32; the probabilities are rounded to the operands' type for the second
// contraction (their sum is taken before that rounding), the result is rounded once.  A row that sees no key is zero; one
// that sees a NaN score is NaN.  Maxima pass over a NaN, sums do not: it is a sum of exactly zero that says "nothing seen"
// (whatever was seen weighs at least 1 at its maximum).
//
// windowMmaKernel: the rows of all query heads that share a kv head are packed into one tile of BM = 16 WM rows
// (row = query * G + head of the group), so that grouped heads read K and V once.  The keys that any row of the tile
// sees are numbered 0 .. nv - 1 ("slots"): the sinks, the window's keys, then the drafted ones; nothing in between is
// touched.  A CTA walks its run of slots in tiles of 64 through a ring of cp.async stages; the four warps split a
// tile into WM groups of rows and 4 / WM groups of keys, each with its own running maximum and sum, merged at the
// end through shared memory.  One row tile per kv head is bound by HBM (16 rows: 16 multiply-adds per byte read).
// With few users the slots are split over `splits` CTAs: up to 8 are a cluster and join their parts through its shared
// memory, parts of more go through the workspace and a second kernel.
// Measured: one token for each of 64 users, 32 query / 8 kv heads x 128, window 4096, 16 sinks, bf16: 192 us, 85 % of the
// measured HBM rate; one user, 8 heads x 64, window 1000: 10 us a call from Python, 6 replayed from a graph.
#include "attention_cached.cuh"
#include "common.cuh"

#include <algorithm>
#include <cmath>

namespace ttb {

constexpr int WN_THREADS = 128;
constexpr int WN_KT = 64;    // slots per tile
constexpr int WN_NODES = 64; // most nodes of a tree (one 64-bit mask per node)
constexpr int WN_CLUSTER = 8; // CTAs of a cluster that every GPU of this kind takes

enum WindowMode { kPrompt = 0, kDecode = 1, kTree = 2 };

struct WindowParams {
  int64_t qb, qh, qs, ob, oh, os;         // element strides over batch, head, query
  int64_t kb, kh, ks, vb, vh, vs;         // ... over batch (paged: block), head, position
  const int32_t *table;                   // [users, pages], or null: one dense run of positions per user
  const int32_t *lens;                    // prompt: keys per user (nullable); decode: cur_pos; tree: cached tokens
  const int32_t *parents, *draftLen;      // tree only; draftLen nullable
  int *bad;                               // status flag for a parent that is not an earlier node
  int pages, blockSize, blocks, parentsUsers;
  int batch, nq, heads, kvHeads, G, keys; // keys: most cached positions of a user
  int offset, window, sinks, splits, mode;
  float scaleLog2;                        // scale * log2(e)
  float *pm, *pl, *po;                    // partial results of the splits, when there are more than a cluster's
};

__device__ __forceinline__ uint32_t wnSmem(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void wnCopy16(uint32_t dst, const void *src, bool pred) {
  const int n = pred ? 16 : 0; // size 0 zero-fills the destination and reads nothing
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(n));
}
__device__ __forceinline__ void wnCommit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N> __device__ __forceinline__ void wnWait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ void wnLdm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void wnLdmT(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T> __device__ __forceinline__ void wnMma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void wnMma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void wnMma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t wnPack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t wnPack<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t wnPack<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&v);
}

// Byte offset of the 16-byte chunk c of row r of a [rows][D] 16-bit tile.  The XOR spreads the eight rows that one
// ldmatrix phase reads over all banks (rows shorter than 128 bytes share a 128-byte line, hence the shift).
template <int D> __device__ __forceinline__ uint32_t wnOff(int r, int c) {
  constexpr int CPR = D / 8, SHIFT = D >= 64 ? 0 : 1, MASK = CPR >= 8 ? 7 : CPR - 1;
  return static_cast<uint32_t>(r * D * 2 + ((c ^ ((r >> SHIFT) & MASK)) << 4));
}

template <int D> struct WindowTile {
  static constexpr int STAGE = 2 * WN_KT * D * 2;                // K and V of one tile, bytes
  static constexpr int STAGES = D <= 64 ? 4 : (D == 128 ? 3 : 2); // 64 / 96 / 128 KiB in flight
  static constexpr bool QREG = D <= 128;                         // query fragments in registers (D = 256: shared memory)
  static constexpr int smem(int bm) { return STAGES * STAGE + (QREG ? 0 : bm * D * 2); }
};

// What a user's keys look like to the row tile whose positions are pMin .. pMax.
struct WindowSlots {
  int sinkN;    // slots 0 .. sinkN - 1 are the positions 0 .. sinkN - 1
  int start;    // slots sinkN .. cached - 1 are the positions start, start + 1, ...
  int cached;   // slots in the cache
  int total;    // ... plus drafted ones
  __device__ __forceinline__ int position(int slot) const { return slot < sinkN ? slot : start + (slot - sinkN); }
};

template <typename T, int D, int WM>
__global__ void __launch_bounds__(WN_THREADS, D <= 128 ? 2 : 1)
    windowMmaKernel(const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const T *__restrict__ kd,
                    const T *__restrict__ vd, T *__restrict__ out, WindowParams p) {
  using Tile = WindowTile<D>;
  constexpr int BM = 16 * WM, WK = 4 / WM, KW = WN_KT / WK, NT = KW / 8; // rows, key groups, keys and 8-key tiles per warp
  constexpr int CPR = D / 8, ND = D / 8, STAGES = Tile::STAGES;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ const T *rowK[STAGES][WN_KT], *rowV[STAGES][WN_KT]; // source rows of a stage's slots, null: zeros
  __shared__ unsigned long long line[WN_NODES];                  // bit u of line[t]: node u is t or an ancestor of t
  __shared__ int up[WN_NODES];
  __shared__ float partM[4][16], partL[4][16];
  __shared__ float rowM[BM], rowL[BM];                           // of all key groups, for the cluster
  pdlLaunchDependents();
  pdlWait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = lane >> 2, t4 = lane & 3;
  const int wm = warp % WM, wk = warp / WM;
  const int split = blockIdx.x % p.splits, mt = blockIdx.x / p.splits, kvh = blockIdx.y, b = blockIdx.z;
  const int rows = p.nq * p.G; // rows of this (user, kv head); nq * G < 2^31 is checked by the host
  const int r0 = mt * BM;

  // ---- what is visible
  int draft = 0, len, pMin, pMax;
  if (p.mode == kDecode) {
    const int pos = p.lens[b];
    len = pos < 0 ? 0 : (pos >= p.keys ? p.keys : pos + 1);
    pMin = pMax = max(pos, -1);
  } else if (p.mode == kTree) {
    len = min(max(p.lens[b], 0), p.keys);
    draft = p.draftLen ? min(max(p.draftLen[b], 0), p.nq) : p.nq;
    pMin = len;
    pMax = len + p.nq - 1;
  } else {
    pMin = p.offset + r0 / p.G;
    pMax = p.offset + min(r0 + BM - 1, rows - 1) / p.G;
    len = p.lens ? min(max(p.lens[b], 0), p.keys) : p.keys;
    len = min(len, pMax + 1);
  }
  if (p.mode == kTree && r0 >= draft * p.G) return; // only padding nodes: their rows are left as they are
  WindowSlots s;
  s.start = min(max(pMin - p.window + 1, 0), len);
  s.sinkN = min(p.sinks, s.start);
  s.cached = s.sinkN + len - s.start;
  s.total = s.cached + draft;
  const int run = ((s.total + p.splits - 1) / p.splits + WN_KT - 1) / WN_KT * WN_KT;
  // min first: split * run could pass 32 bits only when run is a full tile beyond total, so it is capped in 64 bits
  const int s0 = static_cast<int>(min(static_cast<int64_t>(split) * run, static_cast<int64_t>(s.total)));
  const int s1 = static_cast<int>(min(static_cast<int64_t>(s0) + run, static_cast<int64_t>(s.total)));
  const int tiles = (s1 - s0 + WN_KT - 1) / WN_KT;

  if (p.mode == kTree) { // ancestors by pointer doubling: after round i every line covers 2^i steps up
    if (tid < WN_NODES) {
      int par = -1;
      if (tid < p.nq) {
        par = p.parents[static_cast<int64_t>(p.parentsUsers == 1 ? 0 : b) * p.nq + tid];
        if (par < -1 || par >= tid) { // not an earlier node: reported, and the node hangs on the cached text
          if (tid < draft) *p.bad = 1;
          par = -1;
        }
      }
      up[tid] = par;
      line[tid] = 1ull << tid;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < 6; ++i) {
      unsigned long long m = 0;
      int far = -1;
      if (tid < WN_NODES) {
        const int u = up[tid];
        m = line[tid] | (u >= 0 ? line[u] : 0ull);
        far = u >= 0 ? up[u] : -1;
      }
      __syncthreads();
      if (tid < WN_NODES) {
        line[tid] = m;
        up[tid] = far;
      }
      __syncthreads();
    }
  }

  // ---- loads.  A slot's page is looked up a whole iteration before its row is fetched.
  auto pageOf = [&](int slot) -> int { // physical block of a cached slot (clamped into the cache, as everywhere)
    if (!p.table || slot >= s.cached || slot >= s1) return b;
    const int blk = p.table[static_cast<int64_t>(b) * p.pages + s.position(slot) / p.blockSize];
    return blk < 0 ? 0 : (blk >= p.blocks ? p.blocks - 1 : blk);
  };
  auto setRow = [&](int stage, int i, int slot, int blk) {
    const T *pk = nullptr, *pv = nullptr;
    if (slot < s1) {
      if (slot < s.cached) {
        const int pos = s.position(slot);
        const int at = p.table ? pos % p.blockSize : pos;
        pk = k + blk * p.kb + kvh * p.kh + at * p.ks;
        pv = v + blk * p.vb + kvh * p.vh + at * p.vs;
      } else {
        const int64_t at = ((static_cast<int64_t>(b) * p.nq + (slot - s.cached)) * p.kvHeads + kvh) * D;
        pk = kd + at;
        pv = vd + at;
      }
    }
    rowK[stage][i] = pk;
    rowV[stage][i] = pv;
  };
  const uint32_t base = wnSmem(smem);
  auto fetch = [&](int stage) {
    const uint32_t sk = base + stage * Tile::STAGE, sv = sk + Tile::STAGE / 2;
    const int c = tid % CPR;
#pragma unroll
    for (int i = 0; i < WN_KT * CPR / WN_THREADS; ++i) {
      const int r = tid / CPR + i * (WN_THREADS / CPR);
      const T *pk = rowK[stage][r], *pv = rowV[stage][r];
      const bool live = pk != nullptr;
      wnCopy16(sk + wnOff<D>(r, c), live ? pk + c * 8 : k, live);
      wnCopy16(sv + wnOff<D>(r, c), live ? pv + c * 8 : v, live);
    }
  };

  // Query rows through shared memory into fragments (D <= 128: by way of the last stage, which is filled later).
  const uint32_t sQ = Tile::QREG ? base + (STAGES - 1) * Tile::STAGE : base + STAGES * Tile::STAGE;
  for (int i = tid; i < BM * CPR; i += WN_THREADS) {
    const int r = i / CPR, c = i % CPR, row = r0 + r;
    const bool live = row < rows;
    const T *src = q;
    if (live) src = q + b * p.qb + (static_cast<int64_t>(kvh) * p.G + row % p.G) * p.qh + (row / p.G) * p.qs + c * 8;
    wnCopy16(sQ + wnOff<D>(r, c), src, live);
  }
  wnCommit();
  for (int i = tid; i < (STAGES - 1) * WN_KT; i += WN_THREADS) {
    const int slot = s0 + i;
    setRow(i / WN_KT, i % WN_KT, slot, pageOf(slot));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (i < tiles) fetch(i);
    wnCommit();
  }
  wnWait<STAGES - 1>(); // the queries
  __syncthreads();
  uint32_t qf[Tile::QREG ? D / 16 : 1][4];
  const int mi = lane >> 3;
  const int qRow = wm * 16 + (lane & 7) + ((mi & 1) << 3);
  if (Tile::QREG) {
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) wnLdm(qf[Tile::QREG ? kk : 0], sQ + wnOff<D>(qRow, kk * 2 + (mi >> 1)));
  }
  int nextPage = tid < WN_KT ? pageOf(s0 + (STAGES - 1) * WN_KT + tid) : 0;

  // This thread's two rows (quad and quad + 8 of the warp's sixteen): their positions and ancestors.
  int rp[2];
  unsigned long long rl[2] = {0, 0};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = min(r0 + wm * 16 + quad + 8 * h, rows - 1), qi = row / p.G;
    rp[h] = p.mode == kDecode ? pMin : p.offset + qi;
    if (p.mode == kTree) {
      rl[h] = line[qi];
      rp[h] = len + __popcll(rl[h]) - 1;
    }
  }

  float o[ND][4];
#pragma unroll
  for (int i = 0; i < ND; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

  for (int it = 0; it < tiles; ++it) {
    const int stage = it % STAGES, ahead = it + STAGES - 1;
    if (tid < WN_KT) setRow(ahead % STAGES, tid, s0 + ahead * WN_KT + tid, nextPage);
    wnWait<STAGES - 2>();
    __syncthreads(); // the tile has landed, the row pointers are set, and the stage of tile it - 1 is free
    if (ahead < tiles) fetch(ahead % STAGES);
    wnCommit();
    if (tid < WN_KT) nextPage = pageOf(s0 + (ahead + 1) * WN_KT + tid);
    const uint32_t sk = base + stage * Tile::STAGE, sv = sk + Tile::STAGE / 2;
    const int kBase = wk * KW; // this warp's keys of the tile

    float sc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t qa[4];
      if (Tile::QREG) {
#pragma unroll
        for (int i = 0; i < 4; ++i) qa[i] = qf[Tile::QREG ? kk : 0][i];
      } else {
        wnLdm(qa, sQ + wnOff<D>(qRow, kk * 2 + (mi >> 1)));
      }
#pragma unroll
      for (int np = 0; np < NT / 2; ++np) {
        uint32_t kf[4];
        wnLdm(kf, sk + wnOff<D>(kBase + np * 16 + (lane & 7) + ((mi >> 1) << 3), kk * 2 + (mi & 1)));
        wnMma<T>(sc[2 * np], qa, kf[0], kf[1]);
        wnMma<T>(sc[2 * np + 1], qa, kf[2], kf[3]);
      }
    }
    // ---- mask.  Most tiles are visible to every row and skip it.
    const int first = s0 + it * WN_KT, last = first + WN_KT - 1;
    const int jLo = first >= s.sinkN ? s.position(first) : s.start; // first window position of the tile
    const bool partial = last >= s1 || last >= s.cached || jLo <= pMax - p.window ||
                         (p.mode == kPrompt && s.position(last) > pMin);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[i][e] *= p.scaleLog2;
    if (partial) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int slot = first + kBase + i * 8 + t4 * 2 + (e & 1), h = e >> 1;
          bool seen = slot < s1;
          if (slot < s.cached) {
            const int j = s.position(slot);
            seen = seen && j <= rp[h] && (j > rp[h] - p.window || j < p.sinks);
          } else if (seen) {
            const int u = slot - s.cached, at = len + __popcll(line[u]) - 1;
            seen = ((rl[h] >> u) & 1ull) && (at > rp[h] - p.window || at < p.sinks);
          }
          if (!seen) sc[i][e] = -INFINITY;
        }
    }
    // ---- online softmax, base 2
    float corr[2], ref[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = m[h];
#pragma unroll
      for (int i = 0; i < NT; ++i) mx = fmaxf(mx, fmaxf(sc[i][2 * h], sc[i][2 * h + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      ref[h] = mx == -INFINITY ? 0.0f : mx; // nothing seen yet: exp2 of -inf is 0
      corr[h] = exp2f(m[h] - ref[h]);
      m[h] = mx;
      l[h] *= corr[h];
    }
    uint32_t pf[NT / 2][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float a0 = exp2f(sc[i][0] - ref[0]), a1 = exp2f(sc[i][1] - ref[0]);
      const float b0 = exp2f(sc[i][2] - ref[1]), b1 = exp2f(sc[i][3] - ref[1]);
      l[0] += a0 + a1;
      l[1] += b0 + b1;
      pf[i >> 1][(i & 1) * 2] = wnPack<T>(a0, a1);
      pf[i >> 1][(i & 1) * 2 + 1] = wnPack<T>(b0, b1);
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      o[i][0] *= corr[0];
      o[i][1] *= corr[0];
      o[i][2] *= corr[1];
      o[i][3] *= corr[1];
    }
#pragma unroll
    for (int kk = 0; kk < NT / 2; ++kk) {
#pragma unroll
      for (int np = 0; np < ND / 2; ++np) {
        uint32_t vf[4];
        wnLdmT(vf, sv + wnOff<D>(kBase + kk * 16 + (lane & 7) + ((mi & 1) << 3), np * 2 + (mi >> 1)));
        wnMma<T>(o[2 * np], pf[kk], vf[0], vf[1]);
        wnMma<T>(o[2 * np + 1], pf[kk], vf[2], vf[3]);
      }
    }
  }
  wnWait<0>();
  __syncthreads(); // no copy in flight, every warp done: the stages become the exchange buffer

  // ---- join the key groups and write
  float *xo = reinterpret_cast<float *>(smem); // [WK][BM][D]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (t4 == 0) {
      partM[warp][quad + 8 * h] = m[h];
      partL[warp][quad + 8 * h] = l[h];
    }
    float *dst = xo + (static_cast<size_t>(wk) * BM + wm * 16 + quad + 8 * h) * D;
#pragma unroll
    for (int i = 0; i < ND; ++i) *reinterpret_cast<float2 *>(dst + i * 8 + t4 * 2) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
  }
  __syncthreads();
  const int liveRows = p.mode == kTree ? draft * p.G : rows;
  const bool clustered = p.splits > 1 && p.splits <= WN_CLUSTER;
  for (int i = tid; i < BM * (D / 4); i += WN_THREADS) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4, row = r0 + r;
    if (row >= liveRows) continue;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < WK; ++w) mx = fmaxf(mx, partM[w * WM + r / 16][r % 16]);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float den = 0.0f;
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float mw = partM[w * WM + r / 16][r % 16], lw = partL[w * WM + r / 16][r % 16];
      if (lw == 0.0f) continue; // this group saw nothing of the row
      const float f = exp2f(mw - mx);
      const float4 x = *reinterpret_cast<const float4 *>(xo + (static_cast<size_t>(w) * BM + r) * D + d);
      den += lw * f;
      acc.x = fmaf(x.x, f, acc.x);
      acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z);
      acc.w = fmaf(x.w, f, acc.w);
    }
    const int head = kvh * p.G + row % p.G, qi = row / p.G;
    if (clustered) { // over the first group's part, which only this thread reads
      *reinterpret_cast<float4 *>(xo + static_cast<size_t>(r) * D + d) = acc;
      if (d == 0) {
        rowM[r] = mx;
        rowL[r] = den;
      }
    } else if (p.splits > 1) {
      const int64_t part = ((static_cast<int64_t>(b) * p.nq + qi) * p.heads + head) * p.splits + split;
      *reinterpret_cast<float4 *>(p.po + part * D + d) = acc;
      if (d == 0) {
        p.pm[part] = mx;
        p.pl[part] = den;
      }
    } else {
      const float inv = den == 0.0f ? 0.0f : 1.0f / den;
      uint2 w;
      w.x = wnPack<T>(acc.x * inv, acc.y * inv);
      w.y = wnPack<T>(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2 *>(out + b * p.ob + head * p.oh + qi * p.os + d) = w;
    }
  }
  if (!clustered) return;
  // ---- join the cluster's parts: its CTAs share the elements out
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  auto remote = [](const void *at, int rank) { // the same place in another CTA
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(wnSmem(at)), "r"(rank));
    return a;
  };
  for (int i = tid + split * WN_THREADS; i < BM * (D / 4); i += WN_THREADS * p.splits) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4, row = r0 + r;
    if (row >= liveRows) continue;
    float ms[WN_CLUSTER], ls[WN_CLUSTER], mx = -INFINITY, den = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < WN_CLUSTER; ++c) {
      ms[c] = -INFINITY;
      ls[c] = 0.0f;
      if (c < p.splits) {
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(ms[c]) : "r"(remote(&rowM[r], c)));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(ls[c]) : "r"(remote(&rowL[r], c)));
      }
      mx = fmaxf(mx, ms[c]);
    }
#pragma unroll
    for (int c = 0; c < WN_CLUSTER; ++c) {
      if (ls[c] == 0.0f) continue; // this part saw nothing of the row
      const float f = exp2f(ms[c] - mx);
      float4 x;
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(remote(xo + static_cast<size_t>(r) * D + d, c)));
      den += ls[c] * f;
      acc.x = fmaf(x.x, f, acc.x);
      acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z);
      acc.w = fmaf(x.w, f, acc.w);
    }
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;
    uint2 w;
    w.x = wnPack<T>(acc.x * inv, acc.y * inv);
    w.y = wnPack<T>(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2 *>(out + b * p.ob + (kvh * p.G + row % p.G) * p.oh + (row / p.G) * p.os + d) = w;
  }
  // no CTA leaves while another may still read its memory
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Joins the splits of a row: one warp per row of [batch, nq, heads], each lane four dims at a time.
template <typename T, int D>
__global__ void __launch_bounds__(128) windowJoinKernel(T *__restrict__ out, WindowParams p, int64_t allRows) {
  pdlLaunchDependents();
  pdlWait();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= allRows) return;
  const int head = static_cast<int>(row % p.heads), qi = static_cast<int>(row / p.heads % p.nq), b = static_cast<int>(row / p.heads / p.nq);
  if (p.mode == kTree && p.draftLen && qi >= p.draftLen[b]) return;
  const float *pm = p.pm + row * p.splits, *pl = p.pl + row * p.splits, *po = p.po + row * p.splits * D;
  float mx = -INFINITY;
  for (int s = 0; s < p.splits; ++s) mx = fmaxf(mx, pm[s]);
  float den = 0.0f;
  for (int s = 0; s < p.splits; ++s) den += pl[s] == 0.0f ? 0.0f : pl[s] * exp2f(pm[s] - mx);
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  for (int d = lane * 4; d < D; d += 128) {
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s = 0; s < p.splits; ++s) {
      if (pl[s] == 0.0f) continue; // this part saw nothing of the row
      const float f = exp2f(pm[s] - mx);
      const float4 x = *reinterpret_cast<const float4 *>(po + static_cast<int64_t>(s) * D + d);
      acc.x = fmaf(x.x, f, acc.x);
      acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z);
      acc.w = fmaf(x.w, f, acc.w);
    }
    uint2 w;
    w.x = wnPack<T>(acc.x * inv, acc.y * inv);
    w.y = wnPack<T>(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2 *>(out + b * p.ob + head * p.oh + qi * p.os + d) = w;
  }
}

// The general form for prompts: any float type, any head_dim up to 256, any strides (head_dim contiguous).  One warp
// per query row; 32 keys at a time, each lane the dot product of one key, then the lanes share the value columns.  Nothing is
// shared between rows and neighbouring lanes read whole keys apart: 32 / 8 heads x 128, f32, 2048 tokens, window 512 take 14.7
// ms (1 TFLOP/s).
template <typename T>
__global__ void __launch_bounds__(128)
    windowRowKernel(const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, T *__restrict__ out, WindowParams p, int D) {
  constexpr int MAXC = 8; // value columns per lane
  __shared__ float sq[4][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  if (row >= static_cast<int64_t>(p.batch) * p.heads * p.nq) return;
  const int qi = static_cast<int>(row % p.nq), head = static_cast<int>(row / p.nq % p.heads), b = static_cast<int>(row / p.nq / p.heads);
  const int kvh = head / p.G, at = p.offset + qi;
  const T *qr = q + b * p.qb + head * p.qh + qi * p.qs;
  for (int d = lane; d < D; d += 32) sq[warp][d] = toF32(qr[d]) * p.scaleLog2;
  __syncwarp();
  int len = p.lens ? min(max(p.lens[b], 0), p.keys) : p.keys;
  len = min(len, at + 1);
  WindowSlots s;
  s.start = min(max(at - p.window + 1, 0), len);
  s.sinkN = min(p.sinks, s.start);
  s.cached = s.sinkN + len - s.start;
  const T *kr = k + b * p.kb + kvh * p.kh, *vr = v + b * p.vb + kvh * p.vh;
  float m = -INFINITY, l = 0.0f, acc[MAXC];
#pragma unroll
  for (int c = 0; c < MAXC; ++c) acc[c] = 0.0f;
  for (int s0 = 0; s0 < s.cached; s0 += 32) {
    const int n = min(32, s.cached - s0);
    float x = -INFINITY;
    if (lane < n) {
      const T *key = kr + s.position(s0 + lane) * p.ks;
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot = fmaf(sq[warp][d], toF32(key[d]), dot);
      x = dot;
    }
    float mx = x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mx = fmaxf(mx, m);
    const float ref = mx == -INFINITY ? 0.0f : mx, corr = exp2f(m - ref), e = exp2f(x - ref);
    m = mx;
    float sum = e;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = l * corr + sum;
#pragma unroll
    for (int c = 0; c < MAXC; ++c) acc[c] *= corr;
    for (int i = 0; i < n; ++i) {
      const float w = __shfl_sync(0xffffffffu, e, i);
      const T *val = vr + s.position(s0 + i) * p.vs;
#pragma unroll
      for (int c = 0; c < MAXC; ++c) {
        if (c * 32 + lane < D) acc[c] = fmaf(w, toF32(val[c * 32 + lane]), acc[c]);
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T *orow = out + b * p.ob + head * p.oh + qi * p.os;
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {
    if (c * 32 + lane < D) orow[c * 32 + lane] = fromF32<T>(acc[c] * inv);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------
static int windowRowTile(int64_t rows) { return rows <= 16 ? 1 : (rows <= 32 ? 2 : 4); } // WM

// Into how many parts the keys of a (user, kv head, row tile) are cut.
static int windowSplits(int64_t batch, int64_t kvHeads, int64_t rows, int64_t maxSlots) {
  const int64_t bm = 16 * windowRowTile(rows);
  const int64_t base = batch * kvHeads * ((rows + bm - 1) / bm);
  const int64_t want = (2 * smCount() + base - 1) / base, most = (maxSlots + 127) / 128;
  const int splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, 128})));
  // A cluster's join costs less than a second kernel and its round trip through memory, as long as each of its CTAs has no
  // more than some 512 slots.  Measured, one user, 32 query / 8 kv heads x 128, one cluster of 8 / all splits and a second
  // kernel, us: 1100 slots 14 / 17, 2000 15 / 20, 2500 16 / 22, 4000 21 / 26.
  return splits > WN_CLUSTER && maxSlots <= 4096 ? WN_CLUSTER : splits;
}

// How a tree's rows are computed, from the sizes that its workspace is asked for with.
struct TreePlan {
  bool tall;  // tensor-core kernel with tiles of 128 rows and 128 slots
  int splits; // runs of slots per row tile, a partial result each (1: the result itself)
};
static TreePlan treePlan(int64_t batch, int64_t nodes, int64_t heads, int64_t kvHeads, int64_t dim, int64_t positions) {
  const int64_t rows = nodes * (heads / kvHeads), slots = positions + nodes;
  TreePlan t;
  // The tensor-core kernel reads faster but starts slower (128 KB of ring to fill, tensor memory to claim, a second kernel
  // for the join).  Measured with 8 kv heads x 4, head_dim 128, this kernel / that one, us: 1 user, 2500 tokens, 8 nodes
  // 29 / 21, 4000 tokens, 8 .. 32 nodes 30 .. 36 / 23 .. 35, 7000 tokens 35 / 40; 4 users, 4000 tokens, 8 nodes 36 / 30; 16
  // users, 2500 tokens, 8 nodes 49 / 61, 8192 tokens, 4 nodes 107 / 120, 16 nodes 109 / 177.  Replayed from a graph, 1 kv head
  // x 8, head_dim 128, 8 nodes, the other kernel / this one: 1 user, 4000 tokens 23 / 23, 7000 tokens 32 / 29, 8 users, 7000
  // tokens 34 / 29.  With head_dim 64 the rule comes too early: 8 kv heads x 4, 8 nodes, 1 user, 7000 tokens 19 / 25, 16000
  // tokens 35 / 32, 8 users, 7000 tokens 35 / 45, 40 users, 2500 tokens 56 / 80.
  t.tall = (dim == 64 || dim == 128) && (slots > 4096 || (slots >= 2048 && 2 * batch * kvHeads > smCount()));
  if (!t.tall) {
    t.splits = windowSplits(batch, kvHeads, rows, slots);
    return t;
  }
  // One CTA per SM: waves x (tiles per CTA + 6 for what a CTA costs besides), at the longest possible length.
  const int64_t base = batch * kvHeads * ((rows + 127) / 128), tiles = (slots + 127) / 128;
  int64_t best = 0;
  t.splits = 1;
  for (int64_t s = 1; s <= std::min<int64_t>(64, std::max<int64_t>(1, tiles / 2)); ++s) {
    const int64_t cost = (base * s + smCount() - 1) / smCount() * ((tiles + s - 1) / s + 6);
    if (s == 1 || cost < best) {
      best = cost;
      t.splits = static_cast<int>(s);
    }
  }
  return t;
}

// Partial results in the workspace: none for up to `joined` splits.
static size_t windowPartBytes(int64_t batch, int64_t nq, int64_t heads, int64_t dim, int64_t splits, int joined) {
  if (splits <= joined) return 0;
  return static_cast<size_t>(batch) * nq * heads * splits * (dim + 2) * sizeof(float);
}

static int64_t maxVisible(int64_t keys, int64_t window, int64_t sinks) {
  return window > 0 && window < keys - sinks ? window + sinks : keys;
}

// Joins the p.splits parts of every row.
template <typename T, int D> static int launchWindowJoin(void *out, const WindowParams &p, cudaStream_t st) {
  const int64_t all = static_cast<int64_t>(p.batch) * p.nq * p.heads;
  TTB_CUDA(launchPdl(windowJoinKernel<T, D>, dim3(static_cast<unsigned>((all + 3) / 4)), dim3(128), 0, st, static_cast<T *>(out), p, all));
  countLaunch();
  TTB_LAUNCH_CHECK();
  return TTB_OK;
}

template <typename T, int D, int WM>
static int launchWindowMma(const void *q, const void *k, const void *v, const void *kd, const void *vd, void *out, const WindowParams &p,
                           cudaStream_t st) {
  constexpr int BM = 16 * WM, smem = WindowTile<D>::smem(BM);
  static bool attrSet[64] = {}; // function attributes belong to a device
  int dev = 0;
  TTB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attrSet[dev]) {
    TTB_CUDA(cudaFuncSetAttribute(windowMmaKernel<T, D, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev >= 0 && dev < 64) attrSet[dev] = true;
  }
  const int64_t mts = (static_cast<int64_t>(p.nq) * p.G + BM - 1) / BM;
  TTB_CHECK(mts * p.splits <= 0x7fffffff, "too many query rows");
  dim3 grid(static_cast<unsigned>(mts * p.splits), static_cast<unsigned>(p.kvHeads), static_cast<unsigned>(p.batch));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(WN_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits <= WN_CLUSTER ? p.splits : 1; // the splits of a row tile are neighbours
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdlEnabled() ? 2 : 1;
  TTB_CUDA(cudaLaunchKernelEx(&cfg, windowMmaKernel<T, D, WM>, static_cast<const T *>(q), static_cast<const T *>(k), static_cast<const T *>(v),
                              static_cast<const T *>(kd), static_cast<const T *>(vd), static_cast<T *>(out), p));
  countLaunch();
  TTB_LAUNCH_CHECK();
  return p.splits > WN_CLUSTER ? launchWindowJoin<T, D>(out, p, st) : TTB_OK;
}

template <typename T, int D>
static int windowMmaRows(const void *q, const void *k, const void *v, const void *kd, const void *vd, void *out, const WindowParams &p,
                         cudaStream_t st) {
  switch (windowRowTile(static_cast<int64_t>(p.nq) * p.G)) {
  case 1: return launchWindowMma<T, D, 1>(q, k, v, kd, vd, out, p, st);
  case 2: return launchWindowMma<T, D, 2>(q, k, v, kd, vd, out, p, st);
  default: return launchWindowMma<T, D, 4>(q, k, v, kd, vd, out, p, st);
  }
}

static bool windowMmaDim(int64_t d) { return d == 32 || d == 64 || d == 128 || d == 256; }

template <typename T>
static int windowMma(const void *q, const void *k, const void *v, const void *kd, const void *vd, void *out, int64_t dim, const WindowParams &p,
                     cudaStream_t st) {
  switch (dim) {
  case 32: return windowMmaRows<T, 32>(q, k, v, kd, vd, out, p, st);
  case 64: return windowMmaRows<T, 64>(q, k, v, kd, vd, out, p, st);
  case 128: return windowMmaRows<T, 128>(q, k, v, kd, vd, out, p, st);
  default: return windowMmaRows<T, 256>(q, k, v, kd, vd, out, p, st);
  }
}

// Positions and windows are 32-bit in the kernels; every sum of two of them stays below 2^31.
constexpr int64_t kMaxPosition = int64_t(1) << 29;

// The fields that every form shares; `window` <= 0 stands for none.
static void windowCommon(WindowParams &p, int64_t batch, int64_t nq, int64_t heads, int64_t kvHeads, int64_t keys, int64_t window, int64_t sinks,
                         float scale) {
  p = WindowParams{};
  p.batch = static_cast<int>(batch);
  p.nq = static_cast<int>(nq);
  p.heads = static_cast<int>(heads);
  p.kvHeads = static_cast<int>(kvHeads);
  p.G = static_cast<int>(heads / kvHeads);
  p.keys = static_cast<int>(keys);
  p.window = static_cast<int>(window <= 0 ? 2 * kMaxPosition : std::min(window, 2 * kMaxPosition));
  p.sinks = static_cast<int>(std::min(sinks, 2 * kMaxPosition));
  p.splits = 1;
  p.parentsUsers = 1;
  p.scaleLog2 = scale * 1.4426950408889634f;
}

// Dense or paged cache [blocks, kvHeads, blockSize, dim] (dense: one block per user).
static void windowCache(WindowParams &p, const void *table, int blocks, int blockSize, int pages, int dim) {
  p.table = static_cast<const int32_t *>(table);
  p.blocks = blocks;
  p.blockSize = blockSize;
  p.pages = pages;
  p.ks = p.vs = dim;
  p.kh = p.vh = static_cast<int64_t>(blockSize) * dim;
  p.kb = p.vb = p.kh * p.kvHeads;
}

static int checkCached(int dtype, int batch, int heads, int kv_heads, int blocks, int block_size, int pages, int head_dim, const void *table,
                       int64_t window, int64_t sinks, float scale) {
  TTB_CHECK(batch > 0 && heads > 0 && kv_heads > 0 && blocks > 0 && block_size > 0 && pages > 0 && head_dim > 0, "empty problem");
  TTB_CHECK(heads % kv_heads == 0, "query heads must be a multiple of kv heads");
  TTB_CHECK(batch <= 65535 && kv_heads <= 65535, "batch and kv heads are limited to 65535");
  TTB_CHECK(static_cast<int64_t>(pages) * block_size <= kMaxPosition, "a user's cache is limited to 2^29 positions");
  TTB_CHECK(table || (blocks == batch && pages == 1), "without a page table the cache is [batch, kv_heads, positions, head_dim]");
  TTB_CHECK(window >= 0 && sinks >= 0, "window and sinks must not be negative");
  TTB_CHECK(std::isfinite(scale), "scale must be finite");
  if (dtype != kBF16 && dtype != kF16) {
    setLastError("attention over a cache: bf16 or f16 only");
    return TTB_ERR_UNSUPPORTED;
  }
  if (!windowMmaDim(head_dim)) {
    setLastError("attention over a cache: head_dim must be 32, 64, 128 or 256");
    return TTB_ERR_UNSUPPORTED;
  }
  return TTB_OK;
}

int indexBadFlag(int **flag); // index_ops.cu: the word that ttb_index_status reports
int sdpaWindowTcgen05Try(const void *q, const void *k, const void *v, const void *lens, void *out, int dtype, int64_t batch, int64_t hq,
                         int64_t hkv, int64_t sq, int64_t skv, int64_t dim, const int64_t *qs, const int64_t *ks, const int64_t *vs,
                         const int64_t *os, int offset, int window, int sinks, float scaleLog2, cudaStream_t st);

} // namespace ttb

using namespace ttb;

extern "C" {

int ttb_sdpa_window(const void *q, const void *k, const void *v, const void *kv_lens, void *out, int dtype, int64_t batch, int64_t heads_q,
                    int64_t heads_kv, int64_t seq_q, int64_t seq_kv, int64_t head_dim, const int64_t *q_strides3, const int64_t *k_strides3,
                    const int64_t *v_strides3, const int64_t *out_strides3, int64_t offset, int64_t window, int64_t sinks, float scale,
                    void *stream) {
  TTB_CHECK((seq_q == 0 || (q && out)) && (seq_q == 0 || seq_kv == 0 || (k && v)), "null tensor"); // an empty tensor may have no address
  TTB_CHECK(batch > 0 && heads_q > 0 && heads_kv > 0 && seq_q >= 0 && seq_kv >= 0 && head_dim > 0, "bad extents");
  TTB_CHECK(heads_q % heads_kv == 0, "query heads must be a multiple of kv heads");
  TTB_CHECK(batch <= 65535 && heads_kv <= 65535 && heads_q <= 1 << 20, "batch and kv heads are limited to 65535");
  TTB_CHECK(offset >= 0 && seq_q <= kMaxPosition && seq_kv <= kMaxPosition && offset <= kMaxPosition, "positions are limited to 2^29");
  TTB_CHECK(window >= 1 && sinks >= 0, "window must be positive and sinks not negative");
  TTB_CHECK(std::isfinite(scale), "scale must be finite");
  TTB_CHECK(seq_q * (heads_q / heads_kv) <= 0x7fffff00, "too many query rows per kv head");
  const size_t es = dtypeSize(dtype);
  if (dtype != kBF16 && dtype != kF16 && dtype != kF32) {
    setLastError("sdpa_window: float types only");
    return TTB_ERR_UNSUPPORTED;
  }
  if (head_dim > 256) {
    setLastError("sdpa_window: head_dim is limited to 256");
    return TTB_ERR_UNSUPPORTED;
  }
  TTB_CHECK(alignedTo(es, q, k, v, out) && alignedTo(4, kv_lens), "tensors must be aligned to their elements");
  if (seq_q == 0) return TTB_OK;
  const int64_t qd[3] = {heads_q * seq_q * head_dim, seq_q * head_dim, head_dim}, kd[3] = {heads_kv * seq_kv * head_dim, seq_kv * head_dim, head_dim};
  const int64_t *qs = q_strides3 ? q_strides3 : qd, *ks = k_strides3 ? k_strides3 : kd, *vs = v_strides3 ? v_strides3 : kd,
                *os = out_strides3 ? out_strides3 : qd;
  WindowParams p;
  windowCommon(p, batch, seq_q, heads_q, heads_kv, seq_kv, window, sinks, scale);
  p.mode = kPrompt;
  p.offset = static_cast<int>(offset);
  p.lens = static_cast<const int32_t *>(kv_lens);
  p.qb = qs[0]; p.qh = qs[1]; p.qs = qs[2];
  p.kb = ks[0]; p.kh = ks[1]; p.ks = ks[2];
  p.vb = vs[0]; p.vh = vs[1]; p.vs = vs[2];
  p.ob = os[0]; p.oh = os[1]; p.os = os[2];
  cudaStream_t st = asStream(stream);
  const double seen = double(seq_q) * std::min<double>(double(seq_kv), double(window + sinks));
  ProfScope prof("sdpa_window", 4.0 * batch * heads_q * seen * head_dim,
                 double(es) * batch * head_dim * (2.0 * heads_q * seq_q + 2.0 * heads_kv * seq_kv), st);
  bool vec = dtype != kF32 && windowMmaDim(head_dim) && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out);
  for (int i = 0; i < 3; ++i) vec = vec && qs[i] % 8 == 0 && ks[i] % 8 == 0 && vs[i] % 8 == 0 && os[i] % 8 == 0;
  if (vec) {
    const int rc = sdpaWindowTcgen05Try(q, k, v, kv_lens, out, dtype, batch, heads_q, heads_kv, seq_q, seq_kv, head_dim, qs, ks, vs, os, p.offset,
                                        p.window, p.sinks, p.scaleLog2, st);
    if (rc >= 0) return rc;
    if (dtype == kBF16) return windowMma<__nv_bfloat16>(q, k, v, nullptr, nullptr, out, head_dim, p, st);
    return windowMma<__half>(q, k, v, nullptr, nullptr, out, head_dim, p, st);
  }
  const int64_t rows = batch * heads_q * seq_q;
  TTB_CHECK((rows + 3) / 4 <= 0x7fffffff, "too many query rows");
  const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
  TTB_DISPATCH_FLOAT(dtype, T, windowRowKernel<T><<<grid, 128, 0, st>>>(static_cast<const T *>(q), static_cast<const T *>(k),
                                                                        static_cast<const T *>(v), static_cast<T *>(out), p,
                                                                        static_cast<int>(head_dim)))
  countLaunch();
  TTB_LAUNCH_CHECK();
  return TTB_OK;
}

size_t ttb_sdpa_window_decode_workspace_bytes(int batch, int heads, int kv_heads, int head_dim, int64_t positions, int64_t window,
                                              int64_t sinks) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || positions <= 0 || heads % kv_heads) return 0;
  return windowPartBytes(batch, 1, heads, head_dim, windowSplits(batch, kv_heads, heads / kv_heads, maxVisible(positions, window, sinks)), WN_CLUSTER);
}

int ttb_sdpa_window_decode(const void *q, const void *k, const void *v, const void *page_table, const void *cur_pos, void *out, int dtype,
                           int batch, int heads, int kv_heads, int blocks, int block_size, int pages_per_user, int head_dim, int64_t window,
                           int64_t sinks, float scale, void *workspace, size_t workspace_bytes, void *stream) {
  TTB_CHECK(q && k && v && cur_pos && out, "null tensor");
  const int rc = checkCached(dtype, batch, heads, kv_heads, blocks, block_size, pages_per_user, head_dim, page_table, window, sinks, scale);
  if (rc) return rc;
  TTB_CHECK(window >= 1, "window must be positive");
  TTB_CHECK(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(workspace), "tensors must be 16-byte aligned");
  TTB_CHECK(alignedTo(4, page_table, cur_pos), "tensors must be aligned to their elements");
  const int64_t positions = static_cast<int64_t>(pages_per_user) * block_size;
  WindowParams p;
  windowCommon(p, batch, 1, heads, kv_heads, positions, window, sinks, scale);
  windowCache(p, page_table, blocks, block_size, pages_per_user, head_dim);
  p.mode = kDecode;
  p.lens = static_cast<const int32_t *>(cur_pos);
  p.qb = p.ob = static_cast<int64_t>(heads) * head_dim;
  p.qh = p.oh = head_dim;
  const int64_t slots = maxVisible(positions, window, sinks);
  p.splits = windowSplits(batch, kv_heads, p.G, slots);
  const size_t need = windowPartBytes(batch, 1, heads, head_dim, p.splits, WN_CLUSTER);
  TTB_CHECK(need == 0 || (workspace && workspace_bytes >= need), "workspace too small (see ttb_sdpa_window_decode_workspace_bytes)");
  const int64_t parts = static_cast<int64_t>(batch) * heads * p.splits;
  p.po = static_cast<float *>(workspace);
  p.pm = p.po + parts * head_dim;
  p.pl = p.pm + parts;
  cudaStream_t st = asStream(stream);
  // an upper bound: every user at the end of its window
  ProfScope prof("sdpa_window_decode", 4.0 * batch * heads * double(slots) * head_dim, 4.0 * batch * kv_heads * double(slots) * head_dim, st);
  if (dtype == kBF16) return windowMma<__nv_bfloat16>(q, k, v, nullptr, nullptr, out, head_dim, p, st);
  return windowMma<__half>(q, k, v, nullptr, nullptr, out, head_dim, p, st);
}

size_t ttb_sdpa_tree_workspace_bytes(int batch, int nodes, int heads, int kv_heads, int head_dim, int64_t positions) {
  if (batch <= 0 || nodes <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || positions <= 0 || heads % kv_heads) return 0;
  const TreePlan plan = treePlan(batch, nodes, heads, kv_heads, head_dim, positions);
  return windowPartBytes(batch, nodes, heads, head_dim, plan.splits, plan.tall ? 1 : WN_CLUSTER);
}

int ttb_sdpa_tree(const void *q, const void *k_draft, const void *v_draft, const void *k_cache, const void *v_cache, const void *page_table,
                  const void *cached_lens, const void *parents, const void *draft_lens, void *out, int dtype, int batch, int nodes, int heads,
                  int kv_heads, int blocks, int block_size, int pages_per_user, int head_dim, int parents_users, int64_t window, int64_t sinks,
                  float scale, void *workspace, size_t workspace_bytes, void *stream) {
  TTB_CHECK(q && k_draft && v_draft && k_cache && v_cache && cached_lens && parents && out, "null tensor");
  const int rc = checkCached(dtype, batch, heads, kv_heads, blocks, block_size, pages_per_user, head_dim, page_table, window, sinks, scale);
  if (rc) return rc;
  TTB_CHECK(nodes >= 1 && nodes <= WN_NODES, "a tree has 1 to 64 nodes");
  TTB_CHECK(parents_users == 1 || parents_users == batch, "parents must be [batch or 1, nodes]");
  TTB_CHECK(static_cast<int64_t>(nodes) * (heads / kv_heads) <= 1 << 24, "too many query rows per kv head");
  TTB_CHECK(aligned16(q) && aligned16(k_draft) && aligned16(v_draft) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out) &&
                aligned16(workspace), "tensors must be 16-byte aligned");
  TTB_CHECK(alignedTo(4, page_table, cached_lens, parents, draft_lens), "tensors must be aligned to their elements");
  const int64_t positions = static_cast<int64_t>(pages_per_user) * block_size;
  WindowParams p;
  windowCommon(p, batch, nodes, heads, kv_heads, positions, window, sinks, scale);
  windowCache(p, page_table, blocks, block_size, pages_per_user, head_dim);
  p.mode = kTree;
  p.lens = static_cast<const int32_t *>(cached_lens);
  p.parents = static_cast<const int32_t *>(parents);
  p.parentsUsers = parents_users;
  p.draftLen = static_cast<const int32_t *>(draft_lens);
  p.qb = p.ob = static_cast<int64_t>(nodes) * heads * head_dim;
  p.qs = p.os = static_cast<int64_t>(heads) * head_dim;
  p.qh = p.oh = head_dim;
  // The workspace must not depend on the window (its size is asked for without one), so neither do the splits.
  const TreePlan plan = treePlan(batch, nodes, heads, kv_heads, head_dim, positions);
  p.splits = plan.splits;
  const size_t need = windowPartBytes(batch, nodes, heads, head_dim, p.splits, plan.tall ? 1 : WN_CLUSTER);
  TTB_CHECK(need == 0 || (workspace && workspace_bytes >= need), "workspace too small (see ttb_sdpa_tree_workspace_bytes)");
  const int flagged = indexBadFlag(&p.bad);
  if (flagged) return flagged;
  const int64_t parts = static_cast<int64_t>(batch) * nodes * heads * p.splits;
  p.po = static_cast<float *>(workspace);
  p.pm = p.po + parts * head_dim;
  p.pl = p.pm + parts;
  cudaStream_t st = asStream(stream);
  const double slots = double(maxVisible(positions, window, sinks)) + nodes; // an upper bound
  ProfScope prof("sdpa_tree", 4.0 * batch * nodes * heads * slots * head_dim,
                 4.0 * batch * kv_heads * slots * head_dim + 4.0 * batch * nodes * heads * head_dim, st);
  if (plan.tall && p.scaleLog2 > 0.0f) {
    AcParams a = {};
    a.table = p.table; a.lens = p.lens; a.parents = p.parents; a.draftLen = p.draftLen; a.bad = p.bad;
    a.pages = p.pages; a.blockSize = p.blockSize; a.blocks = p.blocks; a.parentsUsers = p.parentsUsers;
    a.nq = p.nq; a.heads = p.heads; a.kvHeads = p.kvHeads; a.G = p.G; a.keys = p.keys; a.window = p.window; a.sinks = p.sinks;
    a.splits = plan.splits;
    a.fmt = dtype == kBF16 ? 1 : 0;
    a.scaleLog2 = p.scaleLog2;
    a.pm = p.pm; a.pl = p.pl; a.po = p.po;
    const int rc2 = sdpaCachedTcgen05(q, k_cache, v_cache, k_draft, v_draft, out, dtype, head_dim, batch, a, st);
    if (rc2 || p.splits == 1) return rc2;
    if (dtype == kBF16) return head_dim == 64 ? launchWindowJoin<__nv_bfloat16, 64>(out, p, st) : launchWindowJoin<__nv_bfloat16, 128>(out, p, st);
    return head_dim == 64 ? launchWindowJoin<__half, 64>(out, p, st) : launchWindowJoin<__half, 128>(out, p, st);
  }
  if (dtype == kBF16) return windowMma<__nv_bfloat16>(q, k_cache, v_cache, k_draft, v_draft, out, head_dim, p, st);
  return windowMma<__half>(q, k_cache, v_cache, k_draft, v_draft, out, head_dim, p, st);
}

} // extern "C"
