// Sampling from whole rows of logits (ttb_sample_logits).  For a row x of `vocab` logits, temperature T:
//   w_i = exp((x_i - max x) / T)                        weights; NaN and -inf logits have none
//   top-k   the k largest logits stay (equal ones: the lower index first)
//   top-p   of those, in the same order, the shortest prefix whose weight reaches p of their sum
//   min-p   of those, the ones with w_i >= min_p
//   draw    the first i, in index order, at which the running sum of what stayed exceeds u times its total
// A weight below 2^-60 of the largest counts as none.  Weights are computed in f32 (relative error near 2^-21), sums
// of up to 32 of them in f32, everything above in f64 in a fixed order, or as integers where atomics are involved: the
// token does not depend on timing.
//
// The work is to read the row; the floor is one pass over it at HBM speed.  One CTA per row (two rows per SM hide each
// other's latencies), 16 warps, each streaming a run of consecutive indices:
//  * Neither cut sorts the row.  A cut ends at one value ("border") and a number of entries equal to it that stay
//    ("ties").  A sample of the row tells where the border must be; one pass then counts and weighs what lies above
//    an interval [lo, hi) around it and collects the entries inside into shared memory (at most SL_LIST), among which
//    the border is found exactly by repeated 1024-way binning.  If the sample misled, the pass's exact counts bracket
//    the border and the next interval is chosen inside the bracket, so the search always ends.  The first interval is
//    open above and sized for some 2500 entries, which answers most top-k and top-p settings at once and finds the
//    largest logit on the way.
//  * The draw is a search too: the 16 warps weigh 16 consecutive runs, the run that holds u times the total is split
//    among the 16 warps again, until 32 entries are left.
// What bounds it: instruction issue, at some 10 instructions per entry and pass.
#include "common.cuh"

#include <cfloat>

namespace ttb {

constexpr int SL_THREADS = 512;
constexpr int SL_WARPS = SL_THREADS / 32;
constexpr int SL_LIST = 8192;               // entries collected by one pass
constexpr int SL_SAMPLE = 4096;
constexpr int SL_BINS = 1024;               // two per thread
constexpr float SL_FIRST = 2500.0f;         // entries aimed at by the first pass
constexpr float SL_FLOOR = 60.0f;           // octaves below the largest weight that count
constexpr float SL_UNIT = 68719476736.0f;   // 2^36 units to the largest weight: SL_LIST of them in two 32-bit halves
constexpr int SL_HALF = 18;                 // ... of 18 bits each, whose sums stay below 2^31
constexpr int64_t SL_MAX_VOCAB = 1 << 22;
static_assert(SL_BINS == 2 * SL_THREADS && SL_LIST <= 1 << 13, "bins per thread; the halves' sums fit 32 bits");

// What one pass found: entries at and above lo and hi, weight at and above lo and another bound, the largest logit.
struct PassResult {
  double mLo, mFrom;
  unsigned int cLo, cHi;
  float top;
};

struct alignas(16) SampleSmem {
  float listX[SL_LIST];
  float sample[SL_SAMPLE];
  unsigned int count[SL_BINS], massLo[SL_BINS], massHi[SL_BINS];
  double dRed[2][SL_WARPS];
  unsigned long long uRed[2][SL_WARPS], picked[2];
  float fRed[2][SL_WARPS];
  unsigned int cRed[2][SL_WARPS], listN;
  int iRed[SL_WARPS], pickBin[2];
  // the draw's current run and target
  int from, to, ok;
  double target, total;
  unsigned long long equalBefore;
  // results of the search's steps, written by one thread and read by all
  PassResult pass;
  float border, lo, hi;
  unsigned int ties;
  unsigned long long through;
};

template <typename V> __device__ __forceinline__ V slWarpSum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float slWarpMax(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float slWarpMin(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// Inclusive running sum over the lanes.
template <typename V> __device__ __forceinline__ V slWarpScan(V v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V left = __shfl_up_sync(0xffffffffu, v, o);
    if (static_cast<int>(threadIdx.x & 31) >= o) v += left;
  }
  return v;
}

// Weights relative to a reference logit: 2^((x - ref) c).  Difference and product are each rounded once, so a weight 2^-h
// is off by some h 2^-24 of itself.  Entries that must not weigh come as -inf, which any c > 0 makes 0.
struct ExpWeight {
  float ref, c;
  __device__ __forceinline__ float operator()(float x) const {
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"((x - ref) * c));
    return w;
  }
};
// Infinities, by definition: logits of at least `from` weigh 1, the others nothing.
struct FlatWeight {
  float from; // +inf under a largest logit of +inf, the lowest float under an infinite temperature
  __device__ __forceinline__ float operator()(float x) const { return x >= from ? 1.0f : 0.0f; }
};
struct Weigher {
  float ref, c;
  bool flat;
  __device__ __forceinline__ void refer(float to, float heat) {
    ref = to;
    c = fminf(fmaxf(1.4426950408889634f / heat, __int_as_float(1)), 1e30f);
    flat = to == INFINITY || heat == INFINITY;
  }
  // Calls f with the weight function as its argument: the hot loops exist once for each kind.
  template <typename F> __device__ __forceinline__ void with(F &&f) const {
    if (flat) f(FlatWeight{ref == INFINITY ? INFINITY : -FLT_MAX});
    else f(ExpWeight{ref, c});
  }
  __device__ __forceinline__ float operator()(float x) const {
    float w = 0.0f;
    with([&](auto weight) { w = weight(x); });
    return w;
  }
};

// Calls f(x, slot, index) for the entries lo .. hi - 1 of a row and end() after every group, all 32 lanes together.  A
// group is up to 4 16-byte vectors per lane; slot numbers the lane's entries in it.  x is -inf for a lane without an
// entry and for NaN.
template <typename T, typename F, typename E> __device__ __forceinline__ void slForRange(const T *x, int lo, int hi, F &&f, E &&end) {
  constexpr int VEC = 16 / sizeof(T), UN = sizeof(T) == 4 ? 4 : 2;
  const int lane = threadIdx.x & 31;
  if (lo >= hi) return;
  const int skip = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x + lo) & 15)) & 15) / static_cast<int>(sizeof(T));
  const int a = min(lo + skip, hi), nv = (hi - a) / VEC;
  const uint4 *vec = reinterpret_cast<const uint4 *>(x + a);
  const int full = nv / (32 * UN) * (32 * UN); // vectors in whole groups
  for (int v0 = 0; v0 < full; v0 += 32 * UN) {
    uint4 raw[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) raw[u] = __ldg(vec + v0 + u * 32 + lane);
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const T *e = reinterpret_cast<const T *>(&raw[u]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f(fmaxf(toF32(e[i]), -INFINITY), u * VEC + i, a + (v0 + u * 32 + lane) * VEC + i);
    }
    end();
  }
  // what is left: the entries in front of the first vector, then fewer than 32 UN vectors and the entries behind them
  if (lo < a) {
    f(lo + lane < a ? fmaxf(toF32(x[lo + lane]), -INFINITY) : -INFINITY, 0, lo + lane);
    end();
  }
  for (int i0 = a + full * VEC + lane; i0 - lane < hi; i0 += 32 * 8) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = i0 + 32 * u < hi ? toF32(x[i0 + 32 * u]) : -INFINITY;
#pragma unroll
    for (int u = 0; u < 8; ++u) f(fmaxf(v[u], -INFINITY), u, i0 + 32 * u);
    end();
  }
}

// Exclusive sum over the block, in thread order, and the total.
template <typename V> __device__ __forceinline__ V slScan(V v, V *scratch, V &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const V run = slWarpScan(v);
  if (lane == 31) scratch[warp] = run;
  __syncthreads();
  const V sums = slWarpScan(lane < SL_WARPS ? scratch[lane] : V(0));
  total = __shfl_sync(0xffffffffu, sums, SL_WARPS - 1);
  const V before = __shfl_sync(0xffffffffu, sums, warp ? warp - 1 : 0);
  __syncthreads();
  return (warp ? before : V(0)) + run - v;
}

// First index of warp w's run (a multiple of 32; the last run ends at n).
__device__ __forceinline__ int slRun(int n, int w) {
  return w >= SL_WARPS ? n : min(n, static_cast<int>((static_cast<int64_t>(n) * w / SL_WARPS) & ~31ll));
}

// One pass over the row.  Entries in [lo, hi) go to the list (s->listN counts them all, also those that do not fit).
// s->pass gets the entries and (weights) the weight at and above lo and hi, the weight at and above `from`, the largest
// logit.
template <typename T>
__device__ __forceinline__ void slPass(const T *x, int n, SampleSmem *s, const Weigher &weigh, float lo, float hi, float from, bool weights) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) s->listN = 0;
  __syncthreads();
  float top = -INFINITY, fLo = 0.0f, fFrom = 0.0f;
  double mLo = 0.0, mFrom = 0.0;
  unsigned int cHi = 0, hits = 0;
  float keep[16];
  auto collect = [&] { // one allocation for the warp's group
    if (!__any_sync(0xffffffffu, hits)) return;
    const unsigned int mine = __popc(hits), run = slWarpScan(mine);
    unsigned int at = 0;
    if (lane == 31) at = atomicAdd(&s->listN, run);
    at = __shfl_sync(0xffffffffu, at, 31) + run - mine;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (hits & (1u << i)) {
        if (at < SL_LIST) s->listX[at] = keep[i];
        ++at;
      }
    }
    hits = 0;
  };
  auto look = [&](float v, int slot) {
    top = fmaxf(top, v);
    const bool above = v >= lo, far = v >= hi;
    if (far) ++cHi;
    if (above && !far) hits |= 1u << slot;
    keep[slot] = v;
  };
  const int first = slRun(n, warp), last = slRun(n, warp + 1);
  if (!weights) {
    slForRange(x, first, last, [&](float v, int slot, int) { look(v, slot); }, collect);
  } else {
    weigh.with([&](auto weight) {
      slForRange(
          x, first, last,
          [&](float v, int slot, int) {
            const float w = weight(v);
            if (v >= lo) fLo += w;
            if (v >= from) fFrom += w;
            look(v, slot);
          },
          [&] {
            mLo += fLo;
            mFrom += fFrom;
            fLo = fFrom = 0.0f;
            collect();
          });
    });
  }
  mLo = slWarpSum(mLo);
  mFrom = slWarpSum(mFrom);
  top = slWarpMax(top);
  cHi = slWarpSum(cHi);
  if (lane == 0) {
    s->dRed[0][warp] = mLo;
    s->dRed[1][warp] = mFrom;
    s->cRed[0][warp] = cHi;
    s->fRed[0][warp] = top;
  }
  __syncthreads();
  if (warp == 0) {
    const int l = lane % SL_WARPS;
    mLo = s->dRed[0][l];
    mFrom = s->dRed[1][l];
    cHi = s->cRed[0][l];
    top = slWarpMax(s->fRed[0][l]);
#pragma unroll
    for (int o = SL_WARPS / 2; o > 0; o >>= 1) {
      mLo += __shfl_xor_sync(0xffffffffu, mLo, o);
      mFrom += __shfl_xor_sync(0xffffffffu, mFrom, o);
      cHi += __shfl_xor_sync(0xffffffffu, cHi, o);
    }
    if (lane == 0) {
      s->pass.mLo = mLo;
      s->pass.mFrom = mFrom;
      s->pass.cHi = cHi;
      s->pass.cLo = cHi + s->listN;
      s->pass.top = top;
    }
  }
  __syncthreads();
}

// Smallest and largest of v over the block.
__device__ __forceinline__ void slSpan(SampleSmem *s, float &a, float &b) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  a = slWarpMin(a);
  b = slWarpMax(b);
  if (lane == 0) {
    s->fRed[0][warp] = a;
    s->fRed[1][warp] = b;
  }
  __syncthreads();
  a = slWarpMin(s->fRed[0][lane % SL_WARPS]);
  b = slWarpMax(s->fRed[1][lane % SL_WARPS]);
  __syncthreads();
}

// The border among the list's entries: the first `rest` entries in descending order, or (byMass) entries as long as
// the units in front of them are fewer than `rest`.  Leaves s->border, s->ties and s->through, the units of the entries
// that stay.
__device__ __forceinline__ void slSelect(SampleSmem *s, const Weigher &weigh, unsigned int count, bool byMass, unsigned long long rest) {
  auto units = [&](float v) { return __float2ull_rn(weigh(v) * SL_UNIT); };
  float least = INFINITY, most = -INFINITY;
  for (unsigned int i = threadIdx.x; i < count; i += SL_THREADS) {
    least = fminf(least, s->listX[i]);
    most = fmaxf(most, s->listX[i]);
  }
  slSpan(s, least, most);
  unsigned long long through = 0;
  while (least < most) {
    for (int i = threadIdx.x; i < SL_BINS; i += SL_THREADS) s->count[i] = s->massLo[i] = s->massHi[i] = 0;
    __syncthreads();
    // least falls into bin 0 and most into the last one or the one before: every round splits what is left.  A range
    // that overflows is halved twice first; one so narrow that the step overflows still separates its ends.
    const float shrink = most - least < INFINITY ? 1.0f : 0.25f, base = least * shrink, step = (SL_BINS - 1) / (most * shrink - base);
    auto binOf = [&](float v) { return min(static_cast<int>((v * shrink - base) * step), SL_BINS - 1); };
    for (unsigned int i = threadIdx.x; i < count; i += SL_THREADS) {
      const float v = s->listX[i];
      if (v >= least && v <= most) {
        const int bin = binOf(v);
        const unsigned long long w = units(v);
        atomicAdd(&s->count[bin], 1u);
        atomicAdd(&s->massLo[bin], static_cast<unsigned int>(w & ((1u << SL_HALF) - 1u)));
        atomicAdd(&s->massHi[bin], static_cast<unsigned int>(w >> SL_HALF));
      }
    }
    __syncthreads();
    // descending bins: thread t holds bins SL_BINS - 1 - 2t and the one below
    const int b0 = SL_BINS - 1 - 2 * static_cast<int>(threadIdx.x), b1 = b0 - 1;
    auto massOf = [&](int bin) { return (static_cast<unsigned long long>(s->massHi[bin]) << SL_HALF) + s->massLo[bin]; };
    const unsigned long long m0 = massOf(b0), m1 = massOf(b1);
    const unsigned long long v0 = byMass ? m0 : s->count[b0], v1 = byMass ? m1 : s->count[b1];
    unsigned long long all, allMass;
    const unsigned long long before = slScan<unsigned long long>(v0 + v1, s->uRed[0], all);
    const unsigned long long massBefore = slScan<unsigned long long>(m0 + m1, s->uRed[1], allMass);
    // the bin in which the limit is reached; rounding may leave it just beyond everything: then the last one
    const unsigned long long want = rest < all ? rest : all;
    if (before < want && want <= before + v0) {
      s->pickBin[0] = b0;
      s->picked[0] = before;
      s->picked[1] = massBefore;
    } else if (before + v0 < want && want <= before + v0 + v1) {
      s->pickBin[0] = b1;
      s->picked[0] = before + v0;
      s->picked[1] = massBefore + m0;
    }
    if (all == 0 && threadIdx.x == 0) { // nothing weighs anything: the largest value is the border
      s->pickBin[0] = binOf(most);
      s->picked[0] = s->picked[1] = 0;
    }
    __syncthreads();
    const int bin = s->pickBin[0];
    rest = want - s->picked[0];
    through += s->picked[1];
    // the bin's own entries; entries of one value share a bin
    float a = INFINITY, b = -INFINITY;
    for (unsigned int i = threadIdx.x; i < count; i += SL_THREADS) {
      const float v = s->listX[i];
      if (v >= least && v <= most && binOf(v) == bin) {
        a = fminf(a, v);
        b = fmaxf(b, v);
      }
    }
    slSpan(s, a, b);
    least = a;
    most = b;
  }
  unsigned int equal = 0, allEqual;
  for (unsigned int i = threadIdx.x; i < count; i += SL_THREADS) equal += s->listX[i] == least;
  slScan<unsigned int>(equal, s->cRed[0], allEqual);
  if (threadIdx.x == 0) {
    const unsigned long long each = units(least);
    unsigned long long keep = byMass ? (each ? (rest + each - 1) / each : allEqual) : rest;
    keep = keep < 1 ? 1 : (keep > allEqual ? allEqual : keep); // a rounded limit may ask for more than there are
    s->border = least;
    s->ties = static_cast<unsigned int>(keep);
    s->through = through + keep * each;
  }
  __syncthreads();
}

// The next interval for a border inside [below, above): where, by the sample, `want` of the bracket's `have` entries
// (byMass: of its weight) lie above; have <= 0: not known, the sample's estimate is taken.  Leaves s->lo and s->hi;
// lo >= hi: the sample has nothing in the bracket.  Nothing here decides a result, only how soon it is found: f32
// throughout.
__device__ __forceinline__ void slChoose(SampleSmem *s, float c, float below, float above, bool byMass, float want, float have, int n, int samples) {
  float a = INFINITY, b = -INFINITY;
  for (int i = threadIdx.x; i < samples; i += SL_THREADS) {
    const float v = s->sample[i];
    if (v >= below && v < above) {
      a = fminf(a, v);
      b = fmaxf(b, v);
    }
  }
  for (int i = threadIdx.x; i < SL_BINS; i += SL_THREADS) s->count[i] = 0;
  slSpan(s, a, b);
  if (!(a < b) || !(b - a < INFINITY)) { // none, or one value only, or too far apart for bins
    if (threadIdx.x == 0) {
      s->lo = a;
      s->hi = a < INFINITY && !(a < b) ? nextafterf(a, INFINITY) : a;
    }
    __syncthreads();
    return;
  }
  const float step = (SL_BINS - 1) / (b - a), width = (b - a) / (SL_BINS - 1);
  for (int i = threadIdx.x; i < samples; i += SL_THREADS) {
    const float v = s->sample[i];
    if (v >= below && v < above) atomicAdd(&s->count[min(static_cast<int>((v - a) * step + 0.5f), SL_BINS - 1)], 1u);
  }
  __syncthreads();
  const int b0 = SL_BINS - 1 - 2 * static_cast<int>(threadIdx.x), b1 = b0 - 1;
  const float c0 = static_cast<float>(s->count[b0]), c1 = static_cast<float>(s->count[b1]);
  // weights relative to the bracket's largest sample: a sum that stays in range whatever the reference
  float w0 = 1.0f, w1 = 1.0f;
  if (byMass) {
    w0 = exp2f((b0 - (SL_BINS - 1)) * width * c);
    w1 = exp2f((b1 - (SL_BINS - 1)) * width * c);
  }
  float cAll, mAll, qAll;
  slScan<float>(c0 + c1, s->fRed[0], cAll);
  const float m0 = slScan<float>(c0 * w0 + c1 * w1, s->fRed[1], mAll) + c0 * w0, m1 = m0 + c1 * w1;
  const float q0 = slScan<float>(c0 * w0 * w0 + c1 * w1 * w1, s->fRed[0], qAll) + c0 * w0 * w0, q1 = q0 + c1 * w1 * w1;
  const float perSample = static_cast<float>(n) / samples;
  const float target = fminf(fmaxf(want / (have > 0.0f ? have : cAll * perSample), 0.0f), 1.0f);
  // Four standard deviations of the sampled share on both sides, less when that would not fit the list.
  float margin = 4.0f, pad = 1.5f / samples;
  for (int round = 0;; ++round) {
    if (threadIdx.x == 0) {
      s->pickBin[0] = -1;
      s->pickBin[1] = SL_BINS;
    }
    __syncthreads();
    auto spread = [&](float q) {
      return margin * sqrtf(q * (1.0f - target) * (1.0f - target) + fmaxf(qAll - q, 0.0f) * target * target) / mAll + pad;
    };
    const float f0 = m0 / mAll, f1 = m1 / mAll, d0 = spread(q0), d1 = spread(q1);
    // highest bin that surely lies at or below the border, lowest bin that surely lies in front of it
    const int least = f0 >= target + d0 ? b0 : (f1 >= target + d1 ? b1 : -1);
    const int most = f1 <= target - d1 ? b1 : (f0 <= target - d0 ? b0 : SL_BINS);
    const int wl = __reduce_max_sync(0xffffffffu, least), wm = __reduce_min_sync(0xffffffffu, most);
    if ((threadIdx.x & 31) == 0) {
      if (wl >= 0) atomicMax(&s->pickBin[0], wl);
      if (wm < SL_BINS) atomicMin(&s->pickBin[1], wm);
    }
    __syncthreads();
    const int pLo = s->pickBin[0], pHi = s->pickBin[1];
    unsigned int inside = 0, sum;
    if (b0 >= pLo && b0 < pHi) inside += s->count[b0];
    if (b1 >= pLo && b1 < pHi) inside += s->count[b1];
    slScan<unsigned int>(inside, s->cRed[0], sum);
    if (sum * perSample <= 0.8f * SL_LIST || pHi - pLo <= 1 || round == 6) {
      // bin edges lie half a bin below the bins' middles; open ends reach to the bracket's
      if (threadIdx.x == 0) {
        s->lo = pLo < 0 ? below : fmaxf(below, a + (pLo - 0.5f) * width);
        s->hi = pHi >= SL_BINS ? above : fminf(above, a + (pHi - 0.5f) * width);
      }
      __syncthreads();
      return;
    }
    margin *= 0.6f;
    pad = 0.0f;
  }
}

// The draw among the entries above `border` and the first `ties` equal to it, with a weight of at least `low`: weigh
// 16 runs, go into the one that holds u times the total, until 32 entries are left.  False: the total is out of range.
template <typename T>
__device__ __forceinline__ bool slPick(const T *x, int n, SampleSmem *s, const Weigher &weigh, float border, unsigned int ties, float low, double u, int32_t *out,
                                    float *prob) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float wBorder = border > -INFINITY ? weigh(border) : 0.0f;
  const double wEqual = wBorder >= low ? static_cast<double>(wBorder) : 0.0;
  int from = 0, to = n;
  bool whole = true;
  for (;;) {
    const int part = whole ? 0 : (to - from + SL_WARPS - 1) / SL_WARPS;
    const int lo = whole ? slRun(n, warp) : min(to, from + warp * part), hi = whole ? slRun(n, warp + 1) : min(to, lo + part);
    double sum = 0.0;
    float f = 0.0f;
    unsigned int equal = 0;
    weigh.with([&](auto weight) {
      slForRange(
          x, lo, hi,
          [&](float v, int, int) {
            const float w = weight(v);
            if (v > border && !(w < low)) f += w; // an overflowed weight (inf) must show in the total
            if (v == border) ++equal;
          },
          [&] {
            sum += f;
            f = 0.0f;
          });
    });
    sum = slWarpSum(sum);
    equal = slWarpSum(equal);
    if (lane == 0) {
      s->dRed[0][warp] = sum;
      s->cRed[0][warp] = equal;
    }
    __syncthreads();
    if (warp == 0) { // lane w: run w
      const bool mine = lane < SL_WARPS;
      const unsigned long long eq = mine ? s->cRed[0][lane] : 0ull;
      unsigned long long seen = slWarpScan(eq) - eq + (whole ? 0ull : s->equalBefore);
      const unsigned long long stay = seen < ties ? (eq < ties - seen ? eq : ties - seen) : 0ull;
      const double m = mine ? s->dRed[0][lane] + wEqual * static_cast<double>(stay) : 0.0;
      const double run = slWarpScan(m);
      const double total = __shfl_sync(0xffffffffu, run, 31);
      const double target = whole ? u * total : s->target;
      const unsigned int hit = __ballot_sync(0xffffffffu, m > 0.0 && run > target), any = __ballot_sync(0xffffffffu, m > 0.0);
      // none: u = 1, or the last bit of a sum taken in another order: the last run that weighs anything
      const int at = hit ? __ffs(hit) - 1 : (any ? 31 - __clz(any) : SL_WARPS - 1);
      if (lane == at) {
        s->target = target - (run - m);
        s->equalBefore = seen;
        const int nf = whole ? slRun(n, lane) : min(to, from + lane * part);
        s->from = nf;
        s->to = whole ? slRun(n, lane + 1) : min(to, nf + part);
        if (whole) {
          s->total = total;
          s->ok = total > 0.0 && total < 1e300;
        }
      }
    }
    __syncthreads();
    if (!s->ok) return false;
    from = s->from;
    to = s->to;
    whole = false;
    if (to - from <= 32) break;
    __syncthreads();
  }
  if (warp == 0) {
    const int i = from + lane;
    const float v = i < to ? fmaxf(toF32(x[i]), -INFINITY) : -INFINITY;
    const float w = weigh(v);
    const bool equal = i < to && v == border;
    const unsigned int eq = __ballot_sync(0xffffffffu, equal);
    const unsigned long long rank = s->equalBefore + __popc(eq & ((1u << lane) - 1u));
    const double mine = v > border && !(w < low) ? static_cast<double>(w) : (equal && rank < ties ? wEqual : 0.0);
    const double run = slWarpScan(mine);
    const unsigned int hit = __ballot_sync(0xffffffffu, mine > 0.0 && run > s->target), any = __ballot_sync(0xffffffffu, mine > 0.0);
    const int at = hit ? __ffs(hit) - 1 : (any ? 31 - __clz(any) : 0);
    if (lane == at) {
      *out = any ? i : -1;
      if (prob) *prob = any ? static_cast<float>(mine / s->total) : 0.0f;
    }
  }
  return true;
}

// The first of the largest logits.
template <typename T> __device__ __forceinline__ void slGreedy(const T *x, int n, SampleSmem *s, int32_t *out, float *prob) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float top = -INFINITY;
  int at = 0x7fffffff;
  slForRange(x, slRun(n, warp), slRun(n, warp + 1),
             [&](float v, int, int i) {
               if (v > top || (v == top && i < at)) { // a range's ragged ends do not come in order
                 top = v;
                 at = i;
               }
             },
             [] {});
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t2 = __shfl_xor_sync(0xffffffffu, top, o);
    const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
    if (t2 > top || (t2 == top && a2 < at)) {
      top = t2;
      at = a2;
    }
  }
  if (lane == 0) {
    s->fRed[0][warp] = top;
    s->iRed[warp] = at;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < SL_WARPS; ++w) {
      if (s->fRed[0][w] > top) { // later warps hold later indices
        top = s->fRed[0][w];
        at = s->iRed[w];
      }
    }
    *out = top > -INFINITY ? at : -1;
    if (prob) *prob = top > -INFINITY ? 1.0f : 0.0f;
  }
}

template <typename T>
__global__ void __launch_bounds__(SL_THREADS, 2)
    sampleLogitsKernel(const T *__restrict__ logits, const float *__restrict__ uniform, const float *__restrict__ temperature,
                       const int32_t *__restrict__ topK, const float *__restrict__ topP, const float *__restrict__ minP, int32_t *__restrict__ out,
                       float *__restrict__ prob, int64_t vocab, int64_t rowStride) {
  extern __shared__ __align__(16) uint8_t smemRaw[];
  SampleSmem *const s = reinterpret_cast<SampleSmem *>(smemRaw);
  pdlLaunchDependents();
  pdlWait();
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T *x = logits + row * rowStride;
  const int n = static_cast<int>(vocab);
  Weigher weigh;
  out += row;
  if (prob) prob += row;
  const float heat = temperature ? temperature[row] : 1.0f;
  if (!(heat > 0.0f)) {
    slGreedy(x, n, s, out, prob);
    return;
  }
  const int32_t k = topK ? topK[row] : 0;
  const float p = topP ? topP[row] : 1.0f;
  const bool cutK = k > 0 && k < n, cutP = p > 0.0f && p < 1.0f;
  float low = minP && minP[row] > 0.0f && minP[row] <= 1.0f ? minP[row] : 0.0f;
  const double u = fmin(fmax(static_cast<double>(uniform[row]), 0.0), 1.0); // NaN: 0

  // ---- a sample: evenly spaced entries, or all of a short row
  const int samples = min(n, SL_SAMPLE);
  const float stride = static_cast<float>(n) / samples;
  float sTop = -INFINITY, unused = INFINITY;
#pragma unroll
  for (int i = 0; i < SL_SAMPLE / SL_THREADS; ++i) {
    const int e = tid + i * SL_THREADS;
    if (e < samples) {
      const float v = fmaxf(toF32(x[min(n - 1, static_cast<int>(e * stride))]), -INFINITY);
      s->sample[e] = v;
      sTop = fmaxf(sTop, v);
    }
  }
  __syncthreads();
  slSpan(s, unused, sTop);

  // What stays: entries above `border`, and of those equal to it the first `ties` by index.
  float border = -INFINITY;
  unsigned int ties = 0;
  const bool cut = cutK || cutP;
  // Without cuts and a min-p the draw needs no search: weights relative to the sample's largest logit will do, unless
  // that is so small that they overflow.
  bool exactTop = false, search = cut || low > 0.0f || !(sTop > -INFINITY && sTop < INFINITY);
  weigh.refer(sTop, heat);
  for (;;) {
    if (search) {
      // The list holds the entries in [lo, hi); the border of the cut at work lies in [below, above).
      bool first = true, again = false, byMass = false;
      bool ask = cut && n > SL_LIST && sTop > -INFINITY && sTop < INFINITY; // choose an interval first
      float below = fmaxf(sTop - SL_FLOOR / weigh.c, -FLT_MAX), above = INFINITY, floor = below;
      float lo = cut ? -FLT_MAX : INFINITY, hi = INFINITY, want = SL_FIRST, have = 0.0f;
      double total = 0.0, atBelow = 0.0, atAbove = 0.0, limit = 0.0, mLo = 0.0, mHi = 0.0;
      int which = cutK ? 0 : 1, round = 0;
      for (bool done = false; !done;) {
        if (ask) {
          slChoose(s, weigh.c, below, above, byMass, want, have, n, samples);
          float nLo = s->lo, nHi = s->hi;
          if (first) { // open above, so that it finds the largest logit
            nLo = fminf(nLo, sTop);
            nHi = INFINITY;
          } else if (!(nLo < nHi) || round >= 6) {
            // no help from the sample (or it misleads): halve the bracket in the order of the floats
            auto order = [](float v) {
              const int i = __float_as_int(v);
              return i >= 0 ? static_cast<int64_t>(i) : -static_cast<int64_t>(i & 0x7fffffff);
            };
            const int64_t mid = (order(below) + order(above)) >> 1;
            nLo = mid >= 0 ? __int_as_float(static_cast<int>(mid)) : __uint_as_float(0x80000000u | static_cast<uint32_t>(-mid));
            nHi = above;
            if (nLo <= below) {
              nLo = below;
              nHi = nextafterf(below, INFINITY);
            }
          }
          lo = first ? nLo : fmaxf(nLo, below);
          hi = fminf(nHi, above);
        }
        slPass(x, n, s, weigh, lo, hi, first ? -FLT_MAX : hi, cutP);
        const PassResult cur = s->pass;
        const unsigned int listed = s->listN;
        if (first) {
          if (cur.top == -INFINITY) {
            if (tid == 0) {
              *out = -1;
              if (prob) *prob = 0.0f;
            }
            return;
          }
          exactTop = true;
          const double rise = (static_cast<double>(cur.top) - static_cast<double>(sTop)) * weigh.c;
          weigh.refer(cur.top, heat);
          if (cur.top == INFINITY) { // only the infinite ones weigh anything: both cuts count them
            border = FLT_MAX;
            if (cut) {
              if (!again) { // how many are there
                again = true;
                ask = false;
                lo = hi = INFINITY;
                continue;
              }
              border = INFINITY;
              ties = cutK && static_cast<unsigned int>(k) < cur.cHi ? static_cast<unsigned int>(k) : cur.cHi;
              if (cutP) ties = static_cast<unsigned int>(ceil(static_cast<double>(p) * static_cast<double>(ties)));
            }
            break;
          }
          if (!cut) break;
          // From here on weights are relative to the true largest logit; the first pass's are rescaled, or taken again
          // when its reference was so far off that they may have overflowed (or there was none).
          double rescale = 1.0;
          if (!again && cutP) {
            if (!(rise < 60.0)) {
              again = true;
              ask = false;
              continue;
            }
            rescale = exp2(-rise);
          }
          first = false;
          floor = fmaxf(cur.top - SL_FLOOR / weigh.c, -FLT_MAX);
          total = cur.mFrom * rescale;
          mHi = 0.0;
          mLo = cur.mLo * rescale;
          byMass = which == 1;
          limit = byMass ? static_cast<double>(p) * total : static_cast<double>(k);
          below = floor;
          atBelow = byMass ? total : 0.0; // entries: not known yet
        } else {
          mHi = cur.mFrom;
          mLo = cur.mLo;
        }
        __syncthreads(); // everyone has read the pass's result
        ask = true;
        ++round;
        // As long as the list answers: the cut's border, then the next cut.
        while (ask && !done) {
          const double hiAt = byMass ? mHi : static_cast<double>(cur.cHi), loAt = byMass ? mLo : static_cast<double>(cur.cLo);
          bool found = false;
          if (limit > hiAt && limit <= loAt) {
            if (listed <= SL_LIST) {
              const double rest = byMass ? ceil((limit - hiAt) * static_cast<double>(SL_UNIT)) : limit - hiAt;
              slSelect(s, weigh, listed, byMass, static_cast<unsigned long long>(fmax(rest, 1.0)));
              border = s->border;
              ties = s->ties;
              total = mHi + static_cast<double>(s->through) / static_cast<double>(SL_UNIT);
              found = true;
            } else {
              if (lo > below) {
                below = lo;
                atBelow = loAt;
              }
              if (hi < above) {
                above = hi;
                atAbove = hiAt;
              }
              if (above <= nextafterf(below, INFINITY)) { // one value, more often than the list is long
                border = below;
                const double w = static_cast<double>(weigh(below)), each = byMass ? fmax(w, 1e-300) : 1.0;
                const double keep = fmin(fmax(ceil((limit - hiAt) / each), 1.0), static_cast<double>(listed));
                ties = static_cast<unsigned int>(keep);
                total = mHi + keep * w;
                found = true;
              }
            }
          } else if (limit > loAt) { // further down
            if (lo < above) {
              above = lo;
              atAbove = loAt;
            }
            if (above <= floor) found = true; // everything that counts stays
          } else if (hi > below) { // further up
            below = hi;
            atBelow = hiAt;
          }
          if (!found && (above <= below || round >= 100)) { // sums that differ in their last bits left nothing between: here it is
            border = below;
            ties = 0xffffffffu;
            found = true;
          }
          if (!found) break; // another interval
          if (which == 1 || !cutP) {
            done = true;
          } else { // top-p next, among what top-k left
            which = 1;
            byMass = true;
            limit = static_cast<double>(p) * total;
            below = floor;
            above = INFINITY;
            atBelow = total;
            atAbove = 0.0;
            round = 0;
          }
        }
        want = static_cast<float>(limit - atAbove);
        have = atBelow > 0.0 ? fmaxf(static_cast<float>(atBelow - atAbove), 1e-30f) : 0.0f;
      }
      if (cut && weigh.ref < INFINITY && border < floor) {
        border = floor;
        ties = 0xffffffffu;
      }
      low *= weigh(weigh.ref);
    }
    if (slPick(x, n, s, weigh, border, ties, low, u, out, prob) || exactTop) return;
    search = true; // nothing was cut, and the sample's largest logit was too small a reference
    __syncthreads();
  }
}

} // namespace ttb

using namespace ttb;

template <typename T>
static int launchSample(const void *logits, const void *uniform, const void *temperature, const void *top_k, const void *top_p, const void *min_p,
                        void *out, void *prob, int64_t rows, int64_t vocab, int64_t row_stride, cudaStream_t st) {
  static bool attrSet[64] = {}; // function attributes belong to a device
  int dev = 0;
  TTB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attrSet[dev]) {
    TTB_CUDA(cudaFuncSetAttribute(sampleLogitsKernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(SampleSmem))));
    if (dev >= 0 && dev < 64) attrSet[dev] = true;
  }
  TTB_CUDA(launchPdl(sampleLogitsKernel<T>, dim3(static_cast<unsigned>(rows)), dim3(SL_THREADS), sizeof(SampleSmem), st,
                     static_cast<const T *>(logits), static_cast<const float *>(uniform), static_cast<const float *>(temperature),
                     static_cast<const int32_t *>(top_k), static_cast<const float *>(top_p), static_cast<const float *>(min_p),
                     static_cast<int32_t *>(out), static_cast<float *>(prob), vocab, row_stride));
  countLaunch();
  TTB_LAUNCH_CHECK();
  return TTB_OK;
}

extern "C" {

size_t ttb_sample_logits_workspace_bytes(int64_t rows, int64_t vocab) {
  (void)rows;
  (void)vocab;
  return 0; // everything fits shared memory
}

int ttb_sample_logits(const void *logits, const void *uniform, const void *temperature, const void *top_k, const void *top_p, const void *min_p,
                      void *out, void *prob, int dtype, int64_t rows, int64_t vocab, int64_t row_stride, void *workspace,
                      size_t workspace_bytes, void *stream) {
  TTB_CHECK(rows >= 0 && vocab >= 1, "bad extents");
  TTB_CHECK(vocab <= SL_MAX_VOCAB, "vocab is limited to 2^22");
  TTB_CHECK(rows <= 0x7fffffff, "too many rows");
  TTB_CHECK(row_stride >= vocab || rows <= 1, "rows overlap");
  if (rows == 0) return TTB_OK;
  TTB_CHECK(logits && uniform && out, "null tensor");
  (void)workspace;
  (void)workspace_bytes;
  cudaStream_t st = asStream(stream);
  ProfScope prof("sample_logits", 4.0 * double(rows) * vocab, double(rows) * vocab * dtypeSize(dtype), st);
  TTB_DISPATCH_FLOAT(dtype, T, return launchSample<T>(logits, uniform, temperature, top_k, top_p, min_p, out, prob, rows, vocab, row_stride, st))
  return TTB_OK;
}

} // extern "C"
