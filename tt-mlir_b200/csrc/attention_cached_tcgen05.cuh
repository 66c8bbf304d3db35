// Attention of many rows over a long cache on the 5th-generation tensor cores: the drafted tokens of a tree when nodes x
// grouped heads make tall row tiles (ttb_sdpa_tree; semantics, slots and partial results as in attention_window.cu).
// Part of attention_tcgen05.cu, whose status word it shares.
//
// One CTA owns 128 rows (node, head of the group) of a (user, kv head) and a run of slots, in tiles of 128:
//   warps 0..3    fetch, two of them keys and two values (a key tile is free as soon as its scores are there, long before
//                 its values), each 64 slots of a tile.  32 neighbouring rows of one page come as TMA boxes; otherwise
//                 (pages that end inside, a window's odd start, drafts, the ragged end) the warp looks every row up and
//                 copies it with cp.async into the swizzled operand layout, zeros for a slot that no row sees
//   warps 4..7, 8..11  softmax of the even and of the odd tiles, one row per thread
//   warp 12       issues tcgen05.mma
// Even and odd tiles are two chains of their own (scores, probabilities, output and maximum), so that one chain's softmax
// runs beside the other's products; at the end the odd chain hands its output to the even one through the ring's memory.
// Bound: HBM as long as a tile of keys and values (64 KB at head_dim 128) takes longer to arrive than a chain's round trip.
// Measured (16 users x 31 nodes, 32 query / 8 kv heads x 128, up to 8192 cached tokens in blocks of 64, bf16): 104 us, 62 %
// of the measured HBM rate over the users' own lengths; 128 CTAs on 148 SMs, the longest user sets the time.  Steps: one
// chain 261 (mma.sync), two chains 159, TMA boxes 114, keys and values fetched apart and joined in the CTA 100; two, three
// or four splits per user 118, 129, 133.
#pragma once

#include "attention_cached.cuh"

namespace ttb {

constexpr int AC_THREADS = 512; // four warpgroups: fetch, two softmax, products (and three idle warps)
template <int D> struct AcShape {
  static constexpr int TILE = 128 * D * 2;          // bytes of a Q, K or V tile
  static constexpr int COLS = 128 * 128;            // bytes of its 64-column part
  static constexpr int STAGES = D == 128 ? 3 : 6;   // K and V of one tile each
  static constexpr int LAG = STAGES - 2;            // tiles on their way behind the one handed over; one stage is being used up
  static constexpr int SMEM = TILE + 2 * STAGES * TILE + 1024 /* alignment slack */ + 512 /* barriers: 8 (4 STAGES + 10) */;
  static_assert(2 * STAGES * TILE >= (D + 2) * 128 * 4, "the ring takes one chain's output, maxima and sums");
};

template <typename T, int D>
__global__ void __launch_bounds__(AC_THREADS, 1)
    sdpaCachedTcgen05Kernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV, const T *__restrict__ q,
                            const T *__restrict__ k, const T *__restrict__ v, const T *__restrict__ kd, const T *__restrict__ vd, T *__restrict__ out,
                            AcParams p) {
  using Sh = AcShape<D>;
  constexpr int R = Sh::STAGES, TILE = Sh::TILE, COLS = Sh::COLS, CPR = D / 8;
  extern __shared__ unsigned char smemRaw[];
  __shared__ uint32_t tmemBaseSlot;
  __shared__ int abortFlag;
  __shared__ unsigned long long line[64]; // bit u of line[t]: node u is t or an ancestor of t
  __shared__ int up[64];

  const uint32_t base = (smemU32(smemRaw) + 1023u) & ~1023u;
  const uint32_t sQ = base, sRing = base + TILE, bars = sRing + 2 * R * TILE;
  // full / empty: K tiles' barriers, then V tiles'
  const uint32_t qFull = bars, full = bars + 8, empty = full + 16 * R, sFull = empty + 16 * R, pReady = sFull + 16 /* [chain][half] */,
                 oFull = pReady + 32, handed = oFull + 16;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    abortFlag = 0;
    mbarInit(qFull, 4);
    for (int i = 0; i < 2 * R; ++i) {
      mbarInit(full + 8 * i, 2);
      mbarInit(empty + 8 * i, 1);
    }
    mbarInit(handed, 4);
    for (int i = 0; i < 2; ++i) {
      mbarInit(sFull + 8 * i, 1);
      mbarInit(pReady + 16 * i, 4);
      mbarInit(pReady + 16 * i + 8, 4);
      mbarInit(oFull + 8 * i, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemU32(&tmemBaseSlot)), "r"(AT_TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdlLaunchDependents(); // the prologue above touched no global memory
  pdlWait();

  const int split = blockIdx.x % p.splits, mt = blockIdx.x / p.splits, kvh = blockIdx.y, b = blockIdx.z;
  const int r0 = mt * 128;
  const int len = min(max(p.lens[b], 0), p.keys), draft = p.draftLen ? min(max(p.draftLen[b], 0), p.nq) : p.nq;
  // Slots: the sinks, the window's positions (from behind the sinks on), the drafts.
  const int start = min(max(max(len - p.window + 1, 0), p.sinks), len), sinkN = min(p.sinks, len);
  const int cached = sinkN + len - start, total = cached + draft;
  const int run = ((total + p.splits - 1) / p.splits + 127) / 128 * 128;
  const int s0 = static_cast<int>(min(static_cast<int64_t>(split) * run, static_cast<int64_t>(total)));
  const int s1 = static_cast<int>(min(static_cast<int64_t>(s0) + run, static_cast<int64_t>(total)));
  const bool padding = r0 >= draft * p.G; // only nodes that do not exist: their rows are left as they are
  const int tiles = padding ? 0 : (s1 - s0 + 127) / 128;

  // Ancestors by pointer doubling: after round i every line covers 2^i steps up.
  if (tid < 64) {
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
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
#pragma unroll 1
  for (int i = 0; i < 6; ++i) {
    unsigned long long bits = 0;
    int far = -1;
    if (tid < 64) {
      const int u = up[tid];
      bits = line[tid] | (u >= 0 ? line[u] : 0ull);
      far = u >= 0 ? up[u] : -1;
    }
    __syncthreads();
    if (tid < 64) {
      line[tid] = bits;
      up[tid] = far;
    }
    __syncthreads();
  }
  const uint32_t tmemBase = tmemBaseSlot;
  volatile int *abortP = &abortFlag;

  // Registers per thread: 64 + 2 x 208 + 24 = 504 of the 4 x 128 at launch.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    auto copy = [&](uint32_t dst, const T *src, bool live) {
      const int n = live ? 16 : 0; // size 0 zero-fills the destination and reads nothing
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    };
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    // 32 rows of a tile from row `to` on, one pointer per lane (null: zeros): two (D = 64: four) rows per instruction.
    auto rows = [&](uint32_t tile, int to, const T *mine, const T *any) {
      constexpr int PER = 32 / CPR;
      const int c = lane % CPR;
#pragma unroll 4
      for (int i = 0; i < 32 / PER; ++i) {
        const int from = i * PER + lane / CPR, row = to + from;
        const T *src = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), from));
        copy(tile + (c >> 3) * COLS + row * 128 + (((c & 7) ^ (row & 7)) << 4), src ? src + c * 8 : any, src != nullptr);
      }
    };
    auto handOver = [&](uint32_t bar) { // this thread's copies have landed: visible to the tensor pipe
      fenceProxyAsyncShared();
      __syncwarp();
      if (lane == 0) mbarArrive(bar);
    };
    if (tiles > 0) {
      const int row = r0 + warp * 32 + lane;
      rows(sQ, warp * 32, row < p.nq * p.G ? q + ((static_cast<int64_t>(b) * p.nq + row / p.G) * p.heads + kvh * p.G + row % p.G) * D : nullptr, q);
      commit();
      const int64_t kh = static_cast<int64_t>(p.blockSize) * D, kb = kh * p.kvHeads;
      auto find = [&](int slot, int64_t &at) -> int { // where the slot's row is: 0 nowhere, 1 in the cache, 2 among the drafts
        if (slot >= s1) return 0;
        if (slot < cached) {
          const int pos = slot < sinkN ? slot : start + (slot - sinkN);
          int blk = b, in = pos;
          if (p.table) {
            blk = p.table[static_cast<int64_t>(b) * p.pages + pos / p.blockSize];
            blk = blk < 0 ? 0 : (blk >= p.blocks ? p.blocks - 1 : blk);
            in = pos % p.blockSize;
          }
          at = blk * kb + kvh * kh + static_cast<int64_t>(in) * D;
          return 1;
        }
        at = ((static_cast<int64_t>(b) * p.nq + (slot - cached)) * p.kvHeads + kvh) * D;
        return 2;
      };
      // 32 slots from `first` on as one box: its block and first row in it, or -1.
      auto box = [&](int first, int &in) -> int {
        if (!p.boxes || first + 32 > min(s1, cached) || (first < sinkN && first + 32 > sinkN)) return -1;
        const int pos = first < sinkN ? first : start + (first - sinkN);
        in = p.table ? pos % p.blockSize : pos;
        if (in + 32 > p.blockSize) return -1;
        if (!p.table) return b;
        const int blk = p.table[static_cast<int64_t>(b) * p.pages + pos / p.blockSize];
        return blk < 0 ? 0 : (blk >= p.blocks ? p.blocks - 1 : blk);
      };
      const bool value = warp >= 2;
      const int to = (warp & 1) * 64; // this warp's rows of a tile
      const CUtensorMap *map = value ? &mapV : &mapK;
      const T *cache = value ? v : k, *drafts = value ? vd : kd;
      const uint32_t fullB = full + (value ? 8 * R : 0), emptyB = empty + (value ? 8 * R : 0);
      int in[2] = {0, 0}, blk[2];
      for (int h = 0; h < 2; ++h) blk[h] = box(s0 + to + 32 * h, in[h]);
      uint32_t arrived = 0; // bit i: the tile i steps back had boxes only, and has been signalled
      int stage = 0, phase = 0;
      for (int j = 0; j < tiles + Sh::LAG; ++j) {
        arrived <<= 1;
        if (j < tiles) {
          if (!__all_sync(0xffffffffu, mbarWait(emptyB + 8 * stage, phase ^ 1, abortP, 1))) break;
          const uint32_t tile = sRing + (2 * stage + (value ? 1 : 0)) * TILE, bar = fullB + 8 * stage;
          for (int h = 0; h < 2; ++h) {
            if (blk[h] >= 0) {
              if (lane == 0) { // this warp's arrival is still due, so the phase cannot end before the bytes are expected
                asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(32 * D * 2) : "memory");
                for (int c = 0; c < D / 64; ++c) tmaLoad4d(tile + c * COLS + (to + 32 * h) * 128, map, bar, c * 64, in[h], kvh, blk[h]);
              }
              __syncwarp();
            } else {
              int64_t at = 0;
              const int kind = find(s0 + j * 128 + to + 32 * h + lane, at);
              rows(tile, to + 32 * h, kind == 0 ? nullptr : (kind == 1 ? cache : drafts) + at, cache);
            }
          }
          if (blk[0] >= 0 && blk[1] >= 0) {
            if (lane == 0) mbarArrive(bar);
            arrived |= 1u;
          }
          if (++stage == R) {
            stage = 0;
            phase ^= 1;
          }
          for (int h = 0; h < 2; ++h) blk[h] = j + 1 < tiles ? box(s0 + (j + 1) * 128 + to + 32 * h, in[h]) : -1; // the next tile's pages
        }
        commit();
        if (j == 0) { // the queries came with the first group
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          handOver(qFull);
        }
        if (j >= Sh::LAG) {
          asm volatile("cp.async.wait_group %0;" ::"n"(Sh::LAG) : "memory");
          if (!(arrived >> Sh::LAG & 1u)) handOver(fullB + 8 * ((j - Sh::LAG) % R));
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory"); // no copy outlives the CTA
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int chain = (warp - 4) >> 2, quarter = warp & 3, lrow = quarter * 32 + lane, row = r0 + lrow;
    const int mine = (tiles + 1 - chain) / 2; // tiles of this chain
    const int node = min(row / p.G, p.nq - 1), pos = len + __popcll(line[node]) - 1;
    // Visible slots of this row: the sinks, cached slots from `near` on, and the drafts in `fresh`.
    const int near = sinkN + max(0, pos - p.window + 1 - start);
    unsigned long long fresh = line[node];
    for (unsigned long long rest = fresh; rest; rest &= rest - 1) {
      const int u = __ffsll(static_cast<long long>(rest)) - 1, at = len + __popcll(line[u]) - 1;
      if (at <= pos - p.window && at >= p.sinks) fresh &= ~(1ull << u);
    }
    const int nearMax = sinkN + max(0, len + p.nq - 1 - p.window + 1 - start); // from here on every row sees the cached slots
    const uint32_t laneAddr = tmemBase + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t sAddr = laneAddr + chain * 128, oAddr = laneAddr + 256 + chain * D;
    const float sl2 = p.scaleLog2;
    float ref = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
      const int first = s0 + (2 * i + chain) * 128;
      if (!__all_sync(0xffffffffu, mbarWait(sFull + 8 * chain, i & 1, abortP, 2))) { ok = false; break; }
      tcFenceAfter();
      uint32_t sc[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tcLoad32(sAddr + c * 32, sc[c]);
      tcWaitLd();
      if (first + 128 > s1 || first + 128 > cached || first < nearMax) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int slot = first + c * 32 + e;
            const bool seen = slot < s1 && (slot < cached ? slot < sinkN || slot >= near : (fresh >> (slot - cached)) & 1ull);
            if (!seen) sc[c][e] = 0xff800000u; // -inf
          }
      }
      awSoftmax<T, D>(sc, sAddr, oAddr, sl2, ref, l, [&](int half) {
        if (lane == 0) mbarArrive(pReady + 16 * chain + 8 * half);
      });
    }
    // All products are done (the ring is free) before the odd chain leaves its output there, one column per row.
    for (int c = 0; c < 2; ++c) {
      if (ok && tiles > c && !__all_sync(0xffffffffu, mbarWait(oFull + 8 * c, 0, abortP, 3))) ok = false;
    }
    tcFenceAfter();
    const uint32_t slot = sRing + lrow * 4; // [dim][row], then maxima, sums
    if (ok && chain == 1 && tiles > 1) {
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        tcLoad32(oAddr + c * 32, r);
        tcWaitLd();
#pragma unroll
        for (int i = 0; i < 32; ++i) asm volatile("st.shared.b32 [%0], %1;" ::"r"(slot + (c * 32 + i) * 512), "r"(r[i]) : "memory");
      }
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(slot + D * 512), "f"(ref) : "memory");
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(slot + (D + 1) * 512), "f"(l) : "memory");
      __syncwarp();
      if (lane == 0) mbarArrive(handed);
    }
    if (ok && chain == 0 && !padding) {
      float f0 = 1.0f, f1 = 0.0f;
      if (tiles > 1) {
        if (!__all_sync(0xffffffffu, mbarWait(handed, 0, abortP, 7))) ok = false;
        float ref1, l1;
        asm volatile("ld.shared.b32 %0, [%1];" : "=f"(ref1) : "r"(slot + D * 512));
        asm volatile("ld.shared.b32 %0, [%1];" : "=f"(l1) : "r"(slot + (D + 1) * 512));
        const float both = fmaxf(ref, ref1);
        f0 = l == 0.0f ? 0.0f : fastExp2((ref - both) * sl2);
        f1 = l1 == 0.0f ? 0.0f : fastExp2((ref1 - both) * sl2);
        l = l * f0 + l1 * f1;
        ref = both;
      }
      const bool live = ok && row < draft * p.G;
      const int64_t orow = (static_cast<int64_t>(b) * p.nq + row / p.G) * p.heads + kvh * p.G + row % p.G, part = orow * p.splits + split;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        if (tiles > 0) {
          tcLoad32(oAddr + c * 32, r);
          tcWaitLd();
        }
        if (!live) continue;
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          x[i] = tiles > 0 && f0 != 0.0f ? __uint_as_float(r[i]) * f0 : 0.0f; // a chain that saw nothing of the row does not count
          if (f1 != 0.0f) {
            float o1;
            asm volatile("ld.shared.b32 %0, [%1];" : "=f"(o1) : "r"(slot + (c * 32 + i) * 512));
            x[i] = fmaf(o1, f1, x[i]);
          }
        }
        if (p.splits > 1) {
#pragma unroll
          for (int g = 0; g < 8; ++g) *reinterpret_cast<float4 *>(p.po + part * D + c * 32 + g * 4) = make_float4(x[g * 4], x[g * 4 + 1], x[g * 4 + 2], x[g * 4 + 3]);
        } else {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (l != 0.0f) { // a NaN among them
              w.x = packPair<T>(x[g * 8] * inv, x[g * 8 + 1] * inv);
              w.y = packPair<T>(x[g * 8 + 2] * inv, x[g * 8 + 3] * inv);
              w.z = packPair<T>(x[g * 8 + 4] * inv, x[g * 8 + 5] * inv);
              w.w = packPair<T>(x[g * 8 + 6] * inv, x[g * 8 + 7] * inv);
            }
            *reinterpret_cast<uint4 *>(out + orow * D + c * 32 + g * 8) = w;
          }
        }
      }
      if (live && p.splits > 1) {
        p.pm[part] = ref == -INFINITY ? -INFINITY : ref * sl2;
        p.pl[part] = l;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 24;");
    const int rounds = __shfl_sync(0xffffffffu, tiles, 0);
    if (warp == 12 && rounds > 0) { // the whole warp in step, see awMma
      const uint32_t tmem = __shfl_sync(0xffffffffu, tmemBase, 0);
      auto wait = [&](uint32_t bar, int parity, int where) { return __all_sync(0xffffffffu, mbarWait(bar, parity, abortP, where)) != 0; };
      constexpr uint32_t HIGH = (2u << 29) | (1u << 14) | (1024u >> 4); // as in the prompt kernel
      const uint32_t idS = instrDescF16(p.fmt, 128, 128, 0, 0), idPV = instrDescF16(p.fmt, 128, D, 0, 1);
      auto desc = [](uint32_t low) -> uint64_t { return (static_cast<uint64_t>(HIGH) << 32) | low; };
      const uint32_t qLow = sQ >> 4;
      bool ok = wait(qFull, 0, 4);
      int stage = 0, phase = 0, old = 0, oldPhase = 0; // of tile j, of tile j - 2
      for (int j = 0; ok && j < rounds + 2; ++j) {
        const int chain = j & 1;
        const uint32_t sCol = tmem + chain * 128, oCol = tmem + 256 + chain * D;
        if (j >= 2) { // O += P V of the chain's tile before
          const uint32_t vLow = ((sRing + (2 * old + 1) * TILE) >> 4) | (static_cast<uint32_t>(COLS >> 4) << 16);
          ok = wait(full + 8 * (R + old), oldPhase, 8);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ok = ok && wait(pReady + 16 * chain + 8 * h, ((j - 2) >> 1) & 1, 5);
            if (ok) {
              tcFenceAfter();
#pragma unroll
              for (int ks = 4 * h; ks < 4 * h + 4; ++ks) awMmaTmemA(oCol, sCol + ks * 8, desc(vLow + ks * (2048 >> 4)), idPV, (j >= 4) | (ks > 0));
            }
          }
          if (!ok) break;
          awCommit(empty + 8 * (R + old));
          if (j + 2 > rounds + 1) awCommit(oFull + 8 * chain); // the chain's last tile
          if (++old == R) {
            old = 0;
            oldPhase ^= 1;
          }
        }
        if (j < rounds) {
          ok = wait(full + 8 * stage, phase, 6);
          if (!ok) break;
          const uint32_t kLow = (sRing + 2 * stage * TILE) >> 4;
          tcFenceAfter();
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = ((ks >> 2) * COLS + (ks & 3) * 32) >> 4;
            awMma(sCol, desc(qLow + off), desc(kLow + off), idS, ks > 0);
          }
          awCommit(sFull + 8 * chain);
          awCommit(empty + 8 * stage);
          if (++stage == R) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  }

  drainAborted(abortP);
  tcFenceBefore();
  __syncthreads();
  if (warp == 12) {
    tcFenceAfter();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmemBase), "r"(AT_TMEM_COLS) : "memory");
  }
}

template <typename T, int D>
static int launchCachedTcgen05(const void *q, const void *k, const void *v, const void *kd, const void *vd, void *out, int batch, AcParams p, cudaStream_t st) {
  // The cache as [blocks, kv heads, block size, D] in boxes of 32 rows; without one every row is copied on its own.
  CUtensorMap mapK = {}, mapV = {};
  const int64_t extents[4] = {D, p.blockSize, p.kvHeads, p.blocks}, row = D, head = row * p.blockSize, strides[3] = {row, head, head * p.kvHeads};
  const int boxRows[3] = {32, 1, 1}, dtype = p.fmt ? kBF16 : kF16;
  p.boxes = p.blockSize >= 32 && makeWindowMap(&mapK, k, dtype, extents, strides, boxRows) && makeWindowMap(&mapV, v, dtype, extents, strides, boxRows);
  static bool attrSet[64] = {}; // function attributes belong to a device
  int dev = 0;
  TTB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attrSet[dev]) {
    TTB_CUDA(cudaFuncSetAttribute(sdpaCachedTcgen05Kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, AcShape<D>::SMEM));
    if (dev >= 0 && dev < 64) attrSet[dev] = true;
  }
  const int64_t mts = (static_cast<int64_t>(p.nq) * p.G + 127) / 128;
  TTB_CHECK(mts * p.splits <= 0x7fffffff, "too many query rows");
  dim3 grid(static_cast<unsigned>(mts * p.splits), static_cast<unsigned>(p.kvHeads), static_cast<unsigned>(batch));
  TTB_CUDA(launchPdl(sdpaCachedTcgen05Kernel<T, D>, grid, dim3(AC_THREADS), AcShape<D>::SMEM, st, mapK, mapV,
                     static_cast<const T *>(q), static_cast<const T *>(k), static_cast<const T *>(v), static_cast<const T *>(kd), static_cast<const T *>(vd),
                     static_cast<T *>(out), p));
  countLaunch();
  TTB_LAUNCH_CHECK();
  return TTB_OK;
}

// The tree's rows over p.splits runs of slots: the result itself, or with several runs the partial results of each, which
// the caller joins.  16-bit types, head_dim 64 or 128, a positive scale.
int sdpaCachedTcgen05(const void *q, const void *k, const void *v, const void *kd, const void *vd, void *out, int dtype, int dim, int batch, const AcParams &p,
                      cudaStream_t st) {
  if (dtype == kBF16) {
    return dim == 64 ? launchCachedTcgen05<__nv_bfloat16, 64>(q, k, v, kd, vd, out, batch, p, st) : launchCachedTcgen05<__nv_bfloat16, 128>(q, k, v, kd, vd, out, batch, p, st);
  }
  return dim == 64 ? launchCachedTcgen05<__half, 64>(q, k, v, kd, vd, out, batch, p, st) : launchCachedTcgen05<__half, 128>(q, k, v, kd, vd, out, batch, p, st);
}

} // namespace ttb
