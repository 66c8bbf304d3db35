// Window attention of a prompt on the 5th-generation tensor cores (ttb_sdpa_window for 16-bit operands with head_dim 64
// or 128; semantics in attention_window.cu).  Part of attention_tcgen05.cu, whose status word it shares.
//
// One CTA owns two row tiles A and B of 128 rows; a row is (query, head of the group), Gp heads of a kv head side by
// side, so that 2 * 128 / Gp neighbouring queries share every key tile.  Packing heads also keeps the union of the rows'
// windows short: it is window + 256 / Gp - 1 keys long.  Keys come in tiles of 128, made of two runs of 64 each: first
// the runs that hold the sinks, then the window's from its first key on, whatever its alignment (a TMA row coordinate has
// none), so that nothing but the last run is loaded in vain.
//   warp 0      TMA producer: Q once, then K and V tiles through one ring
//   warp 1      issues tcgen05.mma: S_A = Q_A K^T, S_B = Q_B K^T, O_A += P_A V, O_B += P_B V
//   warps 4..7  softmax of tile A, one row per thread;  warps 8..11 of tile B.  They take over most of the registers of the
//               first four warps (setmaxnreg: 56 + 2 x 224 per thread of each warpgroup = 3 x 168 at launch), which keeps a
//               row's 128 scores in registers without spills.
// While the softmax warps of one tile work, the tensor pipe runs the other tile's two products.  A tile's probabilities
// overwrite the first half of the columns of the scores they come from and are read from there as the A operand; a
// score buffer is rewritten only by a product issued after the one that read its probabilities, so the hand-over needs
// just two barriers per tile and step (scores there; probabilities there).
//   TMEM: S_A 0..127, S_B 128..255, O_A 256.., O_B 256 + D..
//   Shared memory: Q_A | Q_B | ring of K / V tiles | barriers.
// Measured (32 query / 8 kv heads x 16384 tokens, head_dim 128, window 2048, 64 sinks, bf16): 0.605 ms, 0.88 PFLOP/s, 52 %
// of the measured cuBLAS rate (0.54 ms from a warm L2).  With parts switched off, at 0.62 ms: without exponentials, maxima
// and sums 0.54, without the products 0.46, without either (loads, tensor-memory traffic, barriers) 0.33, without the TMA
// loads unchanged.  So neither unit is saturated (the tensor pipe works 48 % of the cycles): a row tile's chain of scores,
// hand-over, softmax, hand-over, values is what it waits for, and two row tiles (tensor memory holds no more) overlap only
// part of it.  Tried and slower: two threads per row with their maxima exchanged (1.35 ms, 96 registers per thread spill),
// exponentials ahead of the maximum (0.76 ms, spills again), hand-overs of 64 keys (0.63 from a warm L2: the score products
// become N = 64); three eighths of the exponentials as polynomials gained less than 1 %.
#pragma once

namespace ttb {

constexpr int AW_THREADS = 384;
constexpr int AW_KEYS = 128;                         // keys per tile
constexpr int AW_RUN = 64;                           // keys per run
template <int D> struct AwShape {
  static constexpr int TILE = 128 * D * 2;           // bytes of a Q, K or V tile
  static constexpr int COLS = 128 * 128;             // bytes of its 64-column part
  static constexpr int RING = D == 128 ? 5 : 8;      // K and V tiles in turn
  static constexpr int SMEM = (2 + RING) * TILE + 1024 /* alignment slack */ + 256 /* barriers */;
};

struct AwParams {
  int heads, kvHeads, G, Gp, Sq, keys;               // keys: extent of k and v that any row can see
  int offset, window, sinks;
  int64_t ob, oh, os;                                // element strides of out over batch, head, query
  const int32_t *lens;
  int fmt;                                           // 1 bf16, 0 f16
  float scaleLog2;
};

// One row's share of a 128-key tile, by one thread: `sc` are its scores (-inf where masked).  `ref` is the maximum the
// exponentials are taken against; it follows the true one only when that has grown by more than a factor 2^8
// (probabilities stay below 2^8), so that most tiles leave O alone.  The probabilities, rounded to T, go over the first
// half of the columns of the scores at sAddr, ready(half) after each half of them; `l` gathers their sum before rounding.
template <typename T, int D, typename Ready>
__device__ __forceinline__ void awSoftmax(uint32_t (&sc)[4][32], uint32_t sAddr, uint32_t oAddr, float sl2, float &ref, float &l, Ready &&ready) {
  float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 32; i += 8)
#pragma unroll
      for (int k = 0; k < 4; ++k) mx4[k] = max3(mx4[k], __uint_as_float(sc[c][i + k]), __uint_as_float(sc[c][i + 4 + k]));
  const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
  float corr = 1.0f;
  if (ref == -INFINITY) {
    ref = mx; // nothing was seen so far: O and l are zero (or NaN)
  } else if ((mx - ref) * sl2 > 8.0f) {
    corr = fastExp2((ref - mx) * sl2);
    ref = mx;
  }
  if (__any_sync(0xffffffffu, corr != 1.0f)) {
    // The scores of this tile were issued behind P V of the one before: O is complete.
    l *= corr;
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t r[32];
      tcLoad32(oAddr + c * 32, r);
      tcWaitLd();
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * corr);
      tcStore32(oAddr + c * 32, r);
    }
  }
  const float negM = ref == -INFINITY ? 0.0f : -ref * sl2;
  const uint64_t sl2x2 = pack2(sl2, sl2), negMx2 = pack2(negM, negM);
  uint64_t sum[2] = {pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t w[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int at = c * 64 + 2 * i;
      float x, y;
      unpack2(fma2(pack2u(sc[at >> 5][at & 31], sc[at >> 5][(at & 31) + 1]), sl2x2, negMx2), x, y);
      x = fastExp2(x);
      y = fastExp2(y);
      sum[i & 1] = add2(sum[i & 1], pack2(x, y));
      w[i] = packPair<T>(x, y);
    }
    tcStore32(sAddr + c * 32, w);
    tcWaitSt();
    tcFenceBefore();
    __syncwarp();
    ready(c);
  }
  float s0, s1, s2, s3;
  unpack2(sum[0], s0, s1);
  unpack2(sum[1], s2, s3);
  l += (s0 + s1) + (s2 + s3);
}

// The products and their commits, called by a whole warp in step; one lane issues.  With the loop around them uniform the
// descriptors can stay in uniform registers (issued from a branch that one lane takes: 567 us instead of 538 for the
// prompt below, from a warm L2).
__device__ __forceinline__ void awMma(uint32_t tmemD, uint64_t descA, uint64_t descB, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p, one;\n\t"
               "elect.sync _|one, 0xffffffff;\n\t"
               "setp.ne.b32 p, %4, 0;\n\t"
               "@one tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(tmemD), "l"(descA), "l"(descB), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void awMmaTmemA(uint32_t tmemD, uint32_t tmemA, uint64_t descB, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p, one;\n\t"
               "elect.sync _|one, 0xffffffff;\n\t"
               "setp.ne.b32 p, %4, 0;\n\t"
               "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(tmemD), "r"(tmemA), "l"(descB), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void awCommit(uint32_t bar) {
  asm volatile("{\n\t.reg .pred one;\n\t"
               "elect.sync _|one, 0xffffffff;\n\t"
               "@one tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
               ::"r"(bar) : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(AW_THREADS, 1)
    sdpaWindowTcgen05Kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK,
                            const __grid_constant__ CUtensorMap mapV, const __grid_constant__ CUtensorMap mapSinkK,
                            const __grid_constant__ CUtensorMap mapSinkV, T *__restrict__ out, AwParams p) {
  using Sh = AwShape<D>;
  constexpr int R = Sh::RING, TILE = Sh::TILE, COLS = Sh::COLS;
  extern __shared__ unsigned char smemRaw[];
  __shared__ uint32_t tmemBaseSlot;
  __shared__ int abortFlag;

  const uint32_t base = (smemU32(smemRaw) + 1023u) & ~1023u;
  const uint32_t sQ = base, sRing = base + 2 * TILE, bars = sRing + R * TILE;
  const uint32_t qFull = bars, full = bars + 8, empty = full + 8 * R, sFull = empty + 8 * R, pReady = sFull + 16 /* [row tile][half] */,
                 oFull = pReady + 32, vClean = oFull + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int perTile = 128 / p.Gp, perCta = 2 * perTile; // queries
  const int groups = p.G / p.Gp, nQ = (p.Sq + perCta - 1) / perCta;
  const int qBlock = blockIdx.x % nQ, rest = blockIdx.x / nQ;
  const int sub = rest % groups, kvh = rest / groups % p.kvHeads, b = rest / groups / p.kvHeads;
  const int q0 = qBlock * perCta, head0 = kvh * p.G + sub * p.Gp;
  const int tilesM = q0 + perTile < p.Sq ? 2 : 1; // row tiles with a query

  if (threadIdx.x == 0) {
    abortFlag = 0;
    mbarInit(qFull, 1);
    for (int i = 0; i < R; ++i) {
      mbarInit(full + 8 * i, 1);
      mbarInit(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbarInit(sFull + 8 * i, 1);
      mbarInit(pReady + 16 * i, 4);
      mbarInit(pReady + 16 * i + 8, 4);
      mbarInit(oFull + 8 * i, 1);
    }
    mbarInit(vClean, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemU32(&tmemBaseSlot)), "r"(AT_TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  const uint32_t tmemBase = tmemBaseSlot;
  pdlLaunchDependents(); // the prologue above touched no global memory
  pdlWait();
  volatile int *abortP = &abortFlag;

  // ---- the CTA's keys: sinks 0 .. sinkN - 1, then start .. n - 1; a window that reaches into the sinks starts behind them
  const int pMin = p.offset + q0, pMax = p.offset + min(q0 + perCta, p.Sq) - 1;
  const int len = p.lens ? min(max(p.lens[b], 0), p.keys) : p.keys;
  const int n = min(len, pMax + 1);
  const int start = min(max(max(pMin - p.window + 1, 0), p.sinks), n), sinkN = min(p.sinks, n);
  const int sinkRuns = (sinkN + AW_RUN - 1) / AW_RUN, runs = sinkRuns + (n - start + AW_RUN - 1) / AW_RUN;
  const int tiles = (runs + 1) / 2;
  // Rows of the last run behind the user's keys hold anything: their values are cleared before the last product.
  const int lastKey0 = runs > sinkRuns ? start + (runs - sinkRuns - 1) * AW_RUN : (runs - 1) * AW_RUN;
  const bool clean = p.lens && runs > 0 && lastKey0 + AW_RUN > len;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      if (lane == 0 && tiles > 0) { // without a key nothing is loaded: no copy may outlive the CTA
        prefetchTensorMap(&mapQ);
        prefetchTensorMap(&mapK);
        prefetchTensorMap(&mapV);
        mbarArriveExpectTx(qFull, tilesM * TILE);
        for (int m = 0; m < tilesM; ++m) {
          for (int c = 0; c < D / 64; ++c) tmaLoad4d(sQ + m * TILE + c * COLS, &mapQ, qFull, c * 64, head0, q0 + m * perTile, b);
        }
        auto load = [&](int seq, int tile, const CUtensorMap *map, const CUtensorMap *sinkMap) -> bool {
          const int s = seq % R, ph = (seq / R) & 1;
          if (!mbarWait(empty + 8 * s, ph ^ 1, abortP, 1)) return false;
          mbarArriveExpectTx(full + 8 * s, TILE);
          for (int h = 0; h < 2; ++h) {
            const int run = 2 * tile + h;
            // a run behind the last one starts behind the tensor: zeros
            const bool sink = run < sinkRuns;
            const int key = sink ? run * AW_RUN : (run < runs ? start + (run - sinkRuns) * AW_RUN : p.keys);
            for (int c = 0; c < D / 64; ++c)
              tmaLoad4d(sRing + s * TILE + c * COLS + h * (COLS / 2), sink ? sinkMap : map, full + 8 * s, c * 64, key, kvh, b);
          }
          return true;
        };
        for (int j = 0; j < tiles; ++j) {
          if (!load(2 * j, j, &mapK, &mapSinkK) || !load(2 * j + 1, j, &mapV, &mapSinkV)) break;
        }
      }
      __syncwarp();
      if (clean) {
        const int seq = 2 * tiles - 1, s = seq % R;
        const bool ok = __all_sync(0xffffffffu, mbarWait(full + 8 * s, (seq / R) & 1, abortP, 2));
        if (ok) {
          const int first = max(0, len - lastKey0), row0 = ((runs - 1) & 1) * AW_RUN;
          for (int i = lane; i < (AW_RUN - first) * 8 * (D / 64); i += 32) {
            const int c = i % 8, col = i / 8 % (D / 64), row = row0 + first + i / 8 / (D / 64);
            const uint32_t at = sRing + s * TILE + col * COLS + row * 128 + c * 16;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
          }
          fenceProxyAsyncShared();
          __syncwarp();
          if (lane == 0) mbarArrive(vClean);
        }
      }
    } else if (warp == 1) {
      const int rounds = __shfl_sync(0xffffffffu, tiles, 0);
      const uint32_t tmem = __shfl_sync(0xffffffffu, tmemBase, 0);
      auto wait = [&](uint32_t bar, int parity, int where) { return __all_sync(0xffffffffu, mbarWait(bar, parity, abortP, where)) != 0; };
      if (rounds > 0) {
        // 32 products per pair of row tiles and key tile leave the issuing lane 64 cycles each: the operand descriptors
        // differ only in the address field of their low word, so each costs one addition (computed in full for every
        // product, the lane took 3300 cycles per key tile and set the pace).
        constexpr uint32_t IDV = (2u << 29) | (1u << 14) | (1024u >> 4); // high word: 128-byte swizzle, version, 1024 bytes per 8 rows
        const uint32_t idS = instrDescF16(p.fmt, 128, AW_KEYS, 0, 0), idPV = instrDescF16(p.fmt, 128, D, 0, 1);
        auto desc = [](uint32_t low) -> uint64_t { return (static_cast<uint64_t>(IDV) << 32) | low; };
        const uint32_t qLow = sQ >> 4, ringLow = sRing >> 4, apart = static_cast<uint32_t>(COLS >> 4) << 16; // V: distance of its 64-column parts
        bool ok = wait(qFull, 0, 3);
        int slot = 0, phase = 0; // of the next tile in the ring
        auto advance = [&] {
          if (++slot == R) {
            slot = 0;
            phase ^= 1;
          }
        };
        for (int j = 0; ok && j <= rounds; ++j) {
          // the ring holds V_{j-1} (from the second round on), then K_j
          const int vSlot = slot;
          if (j > 0) {
            ok = wait(full + 8 * slot, phase, 5);
            if (ok && j == rounds && clean) ok = wait(vClean, 0, 6);
            advance();
          }
          const int kSlot = slot;
          if (ok && j < rounds) {
            ok = wait(full + 8 * slot, phase, 4);
            advance();
          }
          const uint32_t vLow = (ringLow + vSlot * (TILE >> 4)) | apart, kLow = ringLow + kSlot * (TILE >> 4);
          for (int m = 0; ok && m < tilesM; ++m) {
            const uint32_t sCol = tmem + m * AW_KEYS, oCol = tmem + 2 * AW_KEYS + m * D;
            if (j > 0) { // O_m += P_m V: steps of 16 keys as each half of the probabilities arrives; P from tensor memory, V MN-major
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                ok = ok && wait(pReady + 16 * m + 8 * h, (j - 1) & 1, 7);
                if (ok) {
                  tcFenceAfter();
#pragma unroll
                  for (int ks = 4 * h; ks < 4 * h + 4; ++ks) awMmaTmemA(oCol, sCol + ks * 8, desc(vLow + ks * (2048 >> 4)), idPV, (j > 1) | (ks > 0));
                }
              }
              if (!ok) break;
              if (m == tilesM - 1) awCommit(empty + 8 * vSlot);
              if (j == rounds) awCommit(oFull + 8 * m);
            }
            if (j < rounds) { // S_m = Q_m K^T: steps of 16 along d, both operands K-major
              const uint32_t aLow = qLow + m * (TILE >> 4);
              tcFenceAfter();
#pragma unroll
              for (int ks = 0; ks < D / 16; ++ks) {
                const uint32_t off = ((ks >> 2) * COLS + (ks & 3) * 32) >> 4;
                awMma(sCol, desc(aLow + off), desc(kLow + off), idS, ks > 0);
              }
              awCommit(sFull + 8 * m);
              if (m == tilesM - 1) awCommit(empty + 8 * kSlot);
            }
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    if ((warp - 4) >> 2 < tilesM) {
      const int m = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane; // TMEM lanes are reachable by warp id mod 4
      const int qi = q0 + m * perTile + row / p.Gp, pos = p.offset + qi;
      const int tMin = p.offset + q0 + m * perTile, tMax = tMin + perTile - 1; // positions of this row tile
      const uint32_t laneAddr = tmemBase + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t sAddr = laneAddr + m * AW_KEYS, oAddr = laneAddr + 2 * AW_KEYS + m * D;
      const float sl2 = p.scaleLog2;
      float ref = -INFINITY, l = 0.0f;
      bool ok = true;
      for (int j = 0; j < tiles; ++j) {
        if (!__all_sync(0xffffffffu, mbarWait(sFull + 8 * m, j & 1, abortP, 8))) { ok = false; break; }
        tcFenceAfter();
        uint32_t sc[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tcLoad32(sAddr + c * 32, sc[c]);
        // Visible keys of this row in each run, relative to its first key: lo .. hi.
        int lo[2], hi[2];
        bool mask = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int run = 2 * j + h;
          if (run < sinkRuns) {
            lo[h] = 0;
            hi[h] = min(pos, sinkN - 1) - run * AW_RUN;
            mask |= min(tMin, sinkN - 1) < run * AW_RUN + AW_RUN - 1;
          } else if (run < runs) {
            const int key0 = start + (run - sinkRuns) * AW_RUN;
            lo[h] = pos - p.window + 1 - key0;
            hi[h] = min(pos, n - 1) - key0;
            mask |= tMax - p.window + 1 > key0 || min(tMin, n - 1) < key0 + AW_RUN - 1;
          } else {
            lo[h] = 1;
            hi[h] = 0;
            mask = true;
          }
        }
        tcWaitLd();
        if (mask) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int at = (c & 1) * 32 + i;
              if (at < lo[c >> 1] || at > hi[c >> 1]) sc[c][i] = 0xff800000u; // -inf
            }
        }
        awSoftmax<T, D>(sc, sAddr, oAddr, sl2, ref, l, [&](int half) {
          if (lane == 0) mbarArrive(pReady + 16 * m + 8 * half);
        });
      }
      if (ok && tiles > 0 && !__all_sync(0xffffffffu, mbarWait(oFull + 8 * m, 0, abortP, 9))) ok = false;
      if (ok) {
        tcFenceAfter();
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T *orow = out + b * p.ob + (head0 + row % p.Gp) * p.oh + qi * p.os;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          if (tiles > 0) {
            tcLoad32(oAddr + c * 32, r);
            tcWaitLd();
          }
          if (qi < p.Sq) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              uint4 v = make_uint4(0, 0, 0, 0); // a row that sees no key (O may never have been written)
              if (l != 0.0f) { // a NaN among them
                v.x = packPair<T>(__uint_as_float(r[g * 8]) * inv, __uint_as_float(r[g * 8 + 1]) * inv);
                v.y = packPair<T>(__uint_as_float(r[g * 8 + 2]) * inv, __uint_as_float(r[g * 8 + 3]) * inv);
                v.z = packPair<T>(__uint_as_float(r[g * 8 + 4]) * inv, __uint_as_float(r[g * 8 + 5]) * inv);
                v.w = packPair<T>(__uint_as_float(r[g * 8 + 6]) * inv, __uint_as_float(r[g * 8 + 7]) * inv);
              }
              *reinterpret_cast<uint4 *>(orow + c * 32 + g * 8) = v;
            }
          }
        }
      }
    }
  }

  drainAborted(abortP);
  tcFenceBefore();
  __syncthreads();
  if (warp == 1) {
    tcFenceAfter();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmemBase), "r"(AT_TMEM_COLS) : "memory");
  }
}

// 16-bit tensor of 4 dimensions (columns first), 128-byte swizzle, box of 64 columns; a dimension of extent 1 takes any
// stride.  Rows outside a dimension read as zero.
static bool makeWindowMap(CUtensorMap *map, const void *ptr, int dtype, const int64_t *extents4, const int64_t *strides3, const int *box3) {
  EncodeTiledFn fn = encodeTiled();
  if (!fn) return false;
  cuuint64_t dims[4], strides[3];
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box3[0]), static_cast<cuuint32_t>(box3[1]), static_cast<cuuint32_t>(box3[2])};
  cuuint32_t steps[4] = {1, 1, 1, 1};
  for (int i = 0; i < 4; ++i) dims[i] = static_cast<cuuint64_t>(extents4[i]);
  for (int i = 0; i < 3; ++i) {
    if (extents4[i + 1] > 1 && strides3[i] <= 0) return false;
    strides[i] = strides3[i] > 0 ? static_cast<cuuint64_t>(strides3[i]) * 2 : 256;
    if (strides[i] >= (1ull << 40)) return false;
  }
  const CUtensorMapDataType dt = dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return fn(map, dt, 4, const_cast<void *>(ptr), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
static int launchWindowTcgen05(const CUtensorMap *maps, void *out, const AwParams &p, unsigned grid, cudaStream_t st) {
  static bool attrSet[64] = {}; // function attributes belong to a device
  int dev = 0;
  TTB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attrSet[dev]) {
    TTB_CUDA(cudaFuncSetAttribute(sdpaWindowTcgen05Kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, AwShape<D>::SMEM));
    if (dev >= 0 && dev < 64) attrSet[dev] = true;
  }
  TTB_CUDA(launchPdl(sdpaWindowTcgen05Kernel<T, D>, dim3(grid), dim3(AW_THREADS), AwShape<D>::SMEM, st, maps[0], maps[1], maps[2], maps[3],
                     maps[4], static_cast<T *>(out), p));
  countLaunch();
  TTB_LAUNCH_CHECK();
  return TTB_OK;
}

// Returns -1 when the problem is outside what this kernel takes (the caller then uses another one), otherwise a status.
int sdpaWindowTcgen05Try(const void *q, const void *k, const void *v, const void *lens, void *out, int dtype, int64_t batch, int64_t hq,
                         int64_t hkv, int64_t sq, int64_t skv, int64_t dim, const int64_t *qs, const int64_t *ks, const int64_t *vs,
                         const int64_t *os, int offset, int window, int sinks, float scaleLog2, cudaStream_t st) {
  if ((dim != 64 && dim != 128) || (dtype != kBF16 && dtype != kF16) || !(scaleLog2 > 0.0f)) return -1;
  const int64_t seen = std::min<int64_t>(skv, offset + sq); // keys behind the last row are nobody's
  if (seen < 1) return -1;
  AwParams p = {};
  p.heads = static_cast<int>(hq);
  p.kvHeads = static_cast<int>(hkv);
  p.G = static_cast<int>(hq / hkv);
  p.Gp = 1;
  while (p.G % (2 * p.Gp) == 0 && p.Gp < 16) p.Gp *= 2;
  p.Sq = static_cast<int>(sq);
  p.keys = static_cast<int>(seen);
  p.offset = offset;
  p.window = window;
  p.sinks = sinks;
  p.ob = os[0]; p.oh = os[1]; p.os = os[2];
  p.lens = static_cast<const int32_t *>(lens);
  p.fmt = dtype == kBF16 ? 1 : 0;
  p.scaleLog2 = scaleLog2;
  const int64_t perCta = 256 / p.Gp, ctas = (sq + perCta - 1) / perCta * (p.G / p.Gp) * hkv * batch;
  if (ctas > 0x7fffffff) return -1;
  CUtensorMap maps[5];
  const int64_t qe[4] = {dim, hq, sq, batch}, qst[3] = {qs[1], qs[2], qs[0]};
  const int qbox[3] = {p.Gp, 128 / p.Gp, 1}, kbox[3] = {AW_RUN, 1, 1};
  if (!makeWindowMap(&maps[0], q, dtype, qe, qst, qbox)) return -1;
  for (int i = 0; i < 4; ++i) {
    const bool value = i & 1, sink = i >= 2;
    const int64_t *s = value ? vs : ks;
    const int64_t ke[4] = {dim, sink ? std::max<int64_t>(1, std::min<int64_t>(sinks, seen)) : seen, hkv, batch}, kst[3] = {s[2], s[1], s[0]};
    if (!makeWindowMap(&maps[1 + i], value ? v : k, dtype, ke, kst, kbox)) return -1;
  }
  const unsigned grid = static_cast<unsigned>(ctas);
  if (dtype == kBF16) return dim == 64 ? launchWindowTcgen05<__nv_bfloat16, 64>(maps, out, p, grid, st) : launchWindowTcgen05<__nv_bfloat16, 128>(maps, out, p, grid, st);
  return dim == 64 ? launchWindowTcgen05<__half, 64>(maps, out, p, grid, st) : launchWindowTcgen05<__half, 128>(maps, out, p, grid, st);
}

} // namespace ttb
