// Sampling from whole rows of logits (ttb_sample_logits).  For a row x of `vocab` logits, temperature T:
//   w_i = exp((x_i - max x) / T)                        weights; NaN and -inf logits have none
//   top-k   the k largest logits stay (equal ones: the lower index first)
//   top-p   of those, in the same order, the shortest prefix whose weight reaches p of their sum
//   min-p   of those, the ones with w_i >= min_p
//   draw    the first i, in index order, at which the running sum of what stayed exceeds u times its total
// A weight below 2^-60 of the largest may count as none.  Weights are computed in f64 (relative error 2^-38) and summed in
// f64 in a fixed order, or, where atomics are involved, as integers of 2^-36 of the largest among them: the token does not
// depend on timing, and differs from the definition's only where u or p lies within some 2^-36 of a border.
//
// The work is to read the row; the floor is one pass over it at HBM speed.  One CTA per row (two rows per SM hide each
// other's latencies), 16 warps, each streaming a run of consecutive indices:
//  * Neither cut sorts the row.  A cut ends at one value ("border") and a number of entries equal to it that stay
//    ("ties").  A sample of the row tells where the border must be; one pass then counts and weighs what lies above
//    an interval [lo, hi) around it and collects the entries inside into shared memory (some SL_LIST), among which the
//    border is found exactly by repeated 1024-way binning.  If the sample misled, the pass's exact counts bracket the
//    border and the next interval is chosen inside the bracket, so the search always ends.  The first pass also finds
//    the largest logit; its interval is open above and sized for some 2500 entries, which answers most top-k and top-p
//    settings at once, unless top-k is deeper than that.
//  * The draw is a search too: of the warps' runs the one that holds u times the total is split among the warps
//    again, until there is a thread for each entry.  After a cut the last pass knows the runs' weights already.
// Measured, 256 rows of 128000 f32 logits (131 MB, 20 us at HBM speed), us: largest logit 48, no cut 72, top-k 50 70, top-k
// 50 and top-p 0.9 127, top-k 40000 178, top-p 0.99 (flat rows) 250 to 280, everything mixed 230.  With weights of f32 exponentials
// it was 43, 41, 62, 79, 103, 166 and 141, and the tokens were not the definition's (see Weigher).  What bounds it: a pass
// that weighs issues some 35 to 40 instructions per entry, 14 of them f64, and takes some 110 thousand of a row's clocks with
// two rows per SM (one that only compares 50; their reads 38 at HBM speed); the steps between passes, which depend on one
// another and whose instructions are fetched for the first time, 13 (sample), 6 to 12 (choosing an interval), 10 to 25
// (border in the list) and 13 (draw).
#include "common.cuh"

#include <cfloat>

namespace ttb {

constexpr int SL_THREADS = 512;
constexpr int SL_WARPS = SL_THREADS / 32;
constexpr int SL_KEEP = 23;                 // entries a thread can collect in one pass
constexpr int SL_LIST = 5120;               // entries that fit: 10 per thread on average, 24 at any of them once in 40 rows
constexpr int SL_SHORT = 8192;              // rows up to this length fit whole: 16 entries per thread, and one of the ragged ends
constexpr int SL_SAMPLE = 4096;
constexpr int SL_STAGES = 6;                // 16-byte vectors of a thread in flight
constexpr int SL_BINS = 1024;               // two per thread
constexpr float SL_FIRST = 2500.0f;         // entries aimed at by the first pass
constexpr float SL_FLOOR = 60.0f;           // octaves below the largest weight that count
constexpr int SL_UNITS = 36;                // a list's largest weight is at most 2^36 units
constexpr int SL_HALF = 18;                 // ... in two halves, which are summed as unsigned 32-bit numbers
constexpr int SL_SIDE = 4;                  // weights computed side by side (2, 4, 8 of them: 290, 245, 286 us with mixed settings)
constexpr double SL_RISE = 300.0;           // octaves that a logit may lie above the reference, within the 400 that weights reach down to
constexpr int64_t SL_MAX_VOCAB = 1 << 22;
static_assert(SL_BINS == 2 * SL_THREADS, "bins per thread");
static_assert(int64_t(SL_THREADS) * SL_KEEP << SL_HALF < int64_t(1) << 32 && SL_UNITS == 2 * SL_HALF, "the halves' sums fit unsigned 32 bits");

// What one pass found: entries and weight at and above lo and hi, the weight at and above a third bound and of everything,
// the largest logit.
struct PassResult {
  double mLo, mHi, mHigh, mAll;
  unsigned int cLo, cHi;
  float top;
  bool fits; // no thread collected more than it can keep
};

enum { KNOWN_NOTHING, KNOWN_LIST, KNOWN_TOP };

struct alignas(16) SampleSmem {
  union {
    uint4 ring[SL_STAGES][SL_THREADS]; // column t: vectors on their way to thread t
    struct {                           // between the passes
      unsigned int count[SL_BINS], massLo[SL_BINS], massHi[SL_BINS];
    };
  };
  float list[SL_KEEP][SL_THREADS]; // column t: what thread t collected
  float sample[SL_SAMPLE];
  double dRed[4][SL_WARPS];
  unsigned long long uRed[2][SL_WARPS], picked, rest;
  float fRed[2][SL_WARPS];
  unsigned int cRed[2][SL_WARPS];
  int iRed[SL_WARPS], pickBin[2];
  float few[32];
  unsigned int fewN, equal;
  // the draw's current run and target
  int from, to, ok;
  double target, total;
  unsigned int equalBefore;
  // results of the search's steps, written by one thread and read by all
  PassResult pass;
  double runAbove[SL_WARPS]; // per warp's run: the weight at and above hi
  float runTop[SL_WARPS];    // ... and the largest logit
  float border, lo, hi, high;
  unsigned int ties;
  double through;
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

// 2^f = 1 + f q(f) on [-1/2, 1/2], q interpolated in eight Chebyshev nodes: off by at most 2^-38 of itself.
__constant__ double slExp2[8] = {0.69314718055683244,   0.24022650695888503,   0.055504109063258665, 0.0096181291352361396,
                                 0.0013333478473685416, 0.00015403475186530786, 1.5303700711365693e-05, 1.325080551750225e-06};

// Weights relative to a reference logit: 2^((x - ref) c) in f64 (weights of f32 exponentials gave some 8 in 10000 draws from
// flat rows of 128000 another token than the definition's).  The exponent is split into the nearest integer n and f in
// [-1/2, 1/2]; n goes into the exponent's bits.  Logits that weigh less than some 2^-400 are raised to there; above 2^1023
// the bits overflow, so a sum is used only where the largest logit shows that none did (SL_RISE).  A NaN counts as the
// smallest logit; -inf may weigh anything and is compared away.
struct Weigher {
  double ref, c; // c: octaves per unit of a logit
  float least;
  __device__ __forceinline__ void refer(float to, float heat) {
    ref = to;
    // Infinitely hot: every finite logit weighs 1.  Where one step of the logits' own grid is 100 octaves, more change nothing.
    const double step = fmin(static_cast<double>(to) - static_cast<double>(nextafterf(to, -INFINITY)), 2.0282409603651670e31); // FLT_MAX's own: 2^104
    c = fmin(fmax(1.4426950408889634 / static_cast<double>(heat), 1e-300), 100.0 / step);
    least = fmaxf(static_cast<float>(ref - 400.0 / c), -FLT_MAX);
  }
  // N weights side by side, so that a coefficient is fetched once for all of them.
  template <int N> __device__ __forceinline__ void each(const float *x, double *w) const {
    constexpr double MAGIC = 6755399441055744.0; // 1.5 * 2^52: the sum's low word is the nearest integer
    double f[N];
    unsigned int n[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const double d = static_cast<double>(fmaxf(x[i], least)) - ref, m = fma(d, c, MAGIC);
      f[i] = fma(d, c, MAGIC - m);
      n[i] = static_cast<unsigned int>(__double2loint(m)) << 20;
      w[i] = slExp2[7];
    }
#pragma unroll
    for (int k = 6; k >= -1; --k) {
      const double a = k < 0 ? 1.0 : slExp2[k < 0 ? 0 : k];
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = fma(f[i], w[i], a);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __hiloint2double(__double2hiint(w[i]) + static_cast<int>(n[i]), __double2loint(w[i]));
  }
  __device__ __forceinline__ double operator()(float x) const {
    double w;
    each<1>(&x, &w);
    return w;
  }
  __device__ __forceinline__ float octaves() const { return fminf(static_cast<float>(c), 1e30f); }
  // The smallest logit whose weight is at least w (0 < w <= 1).
  __device__ __forceinline__ float reaches(double w) const {
    float x = static_cast<float>(ref + (log2(w) - 1.6e-16) / c); // within a step or two (a weight within 2^-53 of 1 is 1)
    if (!(x > -FLT_MAX)) return -FLT_MAX;
    for (int i = 0; i < 4; ++i) x = nextafterf(x, -INFINITY);
    for (int i = 0; i < 8 && (*this)(x) < w; ++i) x = nextafterf(x, INFINITY);
    return x;
  }
};

// Calls f(v) for entries lo .. hi - 1 of a row, N (4 or 8) of them (an array) per lane at a time, all 32 lanes together; an
// entry that a lane does not have is -inf.  f lets the warp vote on all of them.  The 16-byte vectors of a range are cut
// into steps of 256 entries; the ragged ends come last.  Vectors come through a ring in shared memory that each lane
// fills and reads for itself, which keeps them in flight without registers.
template <int N, typename T, typename F>
__device__ __forceinline__ void slForRange(const T *x, SampleSmem *s, int lo, int hi, F &&f) {
  constexpr int VEC = 16 / sizeof(T), PER = 8 / VEC, AHEAD = SL_STAGES / PER; // entries per vector, vectors per step, steps in flight
  constexpr int TAKE = N < VEC ? N : VEC;
  const int lane = threadIdx.x & 31;
  if (lo >= hi) return;
  const int skip = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x + lo) & 15)) & 15) / static_cast<int>(sizeof(T));
  const int a = min(lo + skip, hi), steps = (hi - a) / 256;
  const uint4 *vec = reinterpret_cast<const uint4 *>(x + a) + lane;
  uint4 *ring = &s->ring[0][threadIdx.x];
  auto fetch = [&](int step, int stage) {
    if (step < steps) {
      const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(ring + stage * (PER * SL_THREADS)));
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst + u * static_cast<uint32_t>(SL_THREADS * sizeof(uint4))),
                     "l"(vec + step * (32 * PER) + u * 32) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) fetch(i, i);
  int stage = 0;
#pragma unroll 1
  for (int c = 0; c < steps; ++c) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(AHEAD - 1) : "memory");
#pragma unroll 2
    for (int u = 0; u < 8; u += N) { // fours are fetched from the ring one after the other: fewer registers
      float v[N];
#pragma unroll
      for (int i0 = 0; i0 < N; i0 += TAKE) {
        struct alignas(TAKE * sizeof(T)) Piece {
          T e[TAKE];
        };
        const Piece raw = *reinterpret_cast<const Piece *>(reinterpret_cast<const T *>(ring + (stage * PER + (u + i0) / VEC) * SL_THREADS) + (u + i0) % VEC);
#pragma unroll
        for (int i = 0; i < TAKE; ++i) v[i0 + i] = toF32(raw.e[i]);
      }
      f(v);
    }
    fetch(c + AHEAD, stage); // this lane has read its column of the stage: it is free
    stage = stage + 1 < AHEAD ? stage + 1 : 0;
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
  // the entries in front of the first vector and behind the last step: fewer than 8 and 256
#pragma unroll 1
  for (int i0 = lo < a ? lo - 128 : a + steps * 256; i0 < hi; i0 = i0 < lo ? a + steps * 256 : i0 + 128) {
    const int from = i0 < lo ? lo : i0, stop = i0 < lo ? a : hi;
    float v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = from + 32 * u + lane < stop ? toF32(x[from + 32 * u + lane]) : -INFINITY;
    f(v);
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

__device__ __forceinline__ float slMax3(float a, float b, float c) { // a NaN counts as absent
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// One pass over the row, a run of it per warp.  Entries in [lo, hi) go to the threads' columns; returns how many this
// thread found (also those that did not fit).  s->pass gets the entries and (WEIGHTS) the weight at and above lo and hi
// and (FIRST) the weight of everything and the largest logit; s->runAbove and s->runTop say the like of each run.  OPEN:
// hi is +inf; otherwise FIRST also weighs what lies at and above `high`.  A step first asks whether any of the lanes'
// entries can lie in the interval, and mostly none does.
template <bool FIRST, bool OPEN, bool WEIGHTS, typename T>
__device__ __forceinline__ unsigned int slPass(const T *row, int n, SampleSmem *s, const Weigher &weigh, float lo, float hi, float high) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float top = -INFINITY, farCount = 0.0f; // farCount stays below 2^24
  double mLo = 0.0, mHi = 0.0, mHigh = 0.0, mAll = 0.0;
  unsigned int mine = 0;
  const float middle = FIRST ? 0.0f : 0.5f * lo + 0.5f * hi, reach = FIRST ? 0.0f : fmaxf(hi - middle, middle - lo) * 1.000001f;
  float *column = &s->list[0][threadIdx.x];
  slForRange<WEIGHTS ? 4 : 8>(row, s, slRun(n, warp), slRun(n, warp + 1), [&](auto &v) {
    constexpr int N = sizeof(v) / sizeof(float);
    bool near;
    if (FIRST) {
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < N; i += 2) m = slMax3(m, v[i], v[i + 1]);
      top = fmaxf(top, m);
      near = m >= lo;
    } else {
      float m = INFINITY; // a NaN (infinite bounds among them) must not hide an entry: the test below is negated
#pragma unroll
      for (int i = 0; i < N; ++i) m = fminf(m, fabsf(v[i] - middle));
      near = !(m > reach);
      float most = -INFINITY;
#pragma unroll
      for (int i = 0; i < N; i += 2) most = slMax3(most, v[i], v[i + 1]);
      if (!__any_sync(0xffffffffu, near || most >= hi)) return; // nothing of interest to anyone
    }
    const bool collect = __any_sync(0xffffffffu, near);
#pragma unroll
    for (int i0 = 0; i0 < N; i0 += SL_SIDE) {
      double w[SL_SIDE];
      if (WEIGHTS) weigh.template each<SL_SIDE>(v + i0, w);
#pragma unroll
      for (int k = 0; k < SL_SIDE; ++k) {
        const float x = v[i0 + k];
        if (WEIGHTS && FIRST && x > -INFINITY) mAll += w[k];
        if (!OPEN && x >= hi) {
          farCount += 1.0f;
          if (WEIGHTS) mHi += w[k];
        }
        if (FIRST && !OPEN && WEIGHTS && x >= high) mHigh += w[k];
      }
      if (!collect) continue;
#pragma unroll
      for (int k = 0; k < SL_SIDE; ++k) {
        const float x = v[i0 + k];
        if (x >= lo && x < hi) {
          if (mine < SL_KEEP) column[mine * SL_THREADS] = x;
          ++mine;
          if (WEIGHTS) mLo += w[k];
        }
      }
    }
  });
  unsigned int cHi = static_cast<unsigned int>(farCount);
  if (WEIGHTS) {
    mHi = OPEN ? 0.0 : slWarpSum(mHi);
    mLo = slWarpSum(mLo) + mHi; // at and above lo
    if (FIRST) mAll = slWarpSum(mAll);
    if (FIRST && !OPEN) mHigh = slWarpSum(mHigh);
  }
  top = slWarpMax(top);
  cHi = slWarpSum(cHi);
  const unsigned int found = slWarpSum(mine);
  const bool full = __any_sync(0xffffffffu, mine > SL_KEEP);
  if (lane == 0) {
    s->dRed[0][warp] = mLo;
    s->dRed[1][warp] = s->runAbove[warp] = mHi;
    s->dRed[2][warp] = mAll;
    s->dRed[3][warp] = mHigh;
    s->cRed[0][warp] = cHi;
    s->cRed[1][warp] = found;
    s->runTop[warp] = top;
    s->iRed[warp] = full;
  }
  __syncthreads();
  if (warp == 0) {
    const int l = lane % SL_WARPS;
    mLo = s->dRed[0][l];
    mHi = s->dRed[1][l];
    mAll = s->dRed[2][l];
    mHigh = s->dRed[3][l];
    cHi = s->cRed[0][l];
    unsigned int listed = s->cRed[1][l];
    top = slWarpMax(s->runTop[l]);
    const bool anyFull = __any_sync(0xffffffffu, s->iRed[l] != 0);
#pragma unroll
    for (int o = SL_WARPS / 2; o > 0; o >>= 1) {
      mLo += __shfl_xor_sync(0xffffffffu, mLo, o);
      mHi += __shfl_xor_sync(0xffffffffu, mHi, o);
      mAll += __shfl_xor_sync(0xffffffffu, mAll, o);
      mHigh += __shfl_xor_sync(0xffffffffu, mHigh, o);
      cHi += __shfl_xor_sync(0xffffffffu, cHi, o);
      listed += __shfl_xor_sync(0xffffffffu, listed, o);
    }
    if (lane == 0) {
      s->pass.mLo = mLo;
      s->pass.mHi = mHi;
      s->pass.mAll = mAll;
      s->pass.mHigh = mHigh;
      s->pass.cHi = cHi;
      s->pass.cLo = cHi + listed;
      s->pass.fits = !anyFull;
      s->pass.top = top;
    }
  }
  __syncthreads();
  return mine;
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

// The border among the collected entries, which lie in [least, most] (this thread holds `count`): the first `limit` in
// descending order, or (byMass) entries as long as the weight in front of them is below `limit`.  Leaves s->border, s->ties
// and (weights) s->through, the weight of the entries that stay.  Weights are taken in units of a power of two that suits the
// largest possible one.
__device__ __forceinline__ void slSelect(SampleSmem *s, const Weigher &weigh, unsigned int count, bool byMass, bool weights, double limit, float least,
                                         float most) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float *column = &s->list[0][threadIdx.x];
  const int shift = min(SL_UNITS - 1 + 1023 - (__double2hiint(weigh(most)) >> 20), 1000); // weigh(most) < 2^SL_UNITS units
  const double unit = __hiloint2double((1023 + shift) << 20, 0);
  auto units = [&](double w) { return __double2ull_rn(w * unit); };
  // f(value, weight) for this thread's entries, SL_SIDE side by side; a value past the last is NaN.
  auto forList = [&](bool weighed, auto &&f) {
#pragma unroll 1
    for (unsigned int i = 0; i < count; i += SL_SIDE) {
      float v[SL_SIDE];
      double w[SL_SIDE];
#pragma unroll
      for (int k = 0; k < SL_SIDE; ++k) v[k] = i + k < count ? column[(i + k) * SL_THREADS] : NAN;
      if (weighed) weigh.template each<SL_SIDE>(v, w);
#pragma unroll
      for (int k = 0; k < SL_SIDE; ++k) f(v[k], weighed ? w[k] : 0.0);
    }
  };
  unsigned long long rest = static_cast<unsigned long long>(fmax(byMass ? ceil(limit * unit) : limit, 1.0));
  for (bool settled = false; !settled;) {
#pragma unroll 1
    for (int i = threadIdx.x; i < SL_BINS; i += SL_THREADS) s->count[i] = s->massLo[i] = s->massHi[i] = 0;
    if (threadIdx.x == 0) s->fewN = 0;
    __syncthreads();
    // A range that overflows is shrunk first; one so narrow that the step overflows still separates its ends.
    const float shrink = most - least < INFINITY ? 1.0f : 0.25f, base = least * shrink, step = (SL_BINS - 1) / (most * shrink - base);
    auto binOf = [&](float v) { return max(0, min(static_cast<int>(fmaf(v, shrink, -base) * step), SL_BINS - 1)); }; // rounded alike in both uses
    forList(byMass, [&](float v, double w) {
      if (v >= least && v <= most) {
        const int bin = binOf(v);
        atomicAdd(&s->count[bin], 1u);
        if (byMass) {
          const unsigned long long u = units(w);
          atomicAdd(&s->massLo[bin], static_cast<unsigned int>(u & ((1u << SL_HALF) - 1u)));
          atomicAdd(&s->massHi[bin], static_cast<unsigned int>(u >> SL_HALF));
        }
      }
    });
    __syncthreads();
    // descending bins: thread t holds bins SL_BINS - 1 - 2t and the one below
    const int b0 = SL_BINS - 1 - 2 * static_cast<int>(threadIdx.x), b1 = b0 - 1;
    auto massOf = [&](int bin) { return (static_cast<unsigned long long>(s->massHi[bin]) << SL_HALF) + s->massLo[bin]; };
    const unsigned int c0 = s->count[b0], c1 = s->count[b1];
    const unsigned long long v0 = byMass ? massOf(b0) : c0, v1 = byMass ? massOf(b1) : c1;
    unsigned long long all;
    const unsigned long long before = slScan<unsigned long long>(v0 + v1, s->uRed[0], all);
    // The bin in which the limit is reached; rounding may leave it just beyond everything: then the last one that holds
    // anything.  Where nothing weighs anything the largest value is the border.
    const unsigned long long want = rest < all ? rest : all;
    const bool at0 = before < want && want <= before + v0, at1 = before + v0 < want && want <= before + v0 + v1;
    if (at0 || at1 || (all == 0 && threadIdx.x == 0)) {
      s->pickBin[0] = at0 ? b0 : (at1 ? b1 : -1);
      s->pickBin[1] = static_cast<int>(at0 ? c0 : (at1 ? c1 : 33u));
      s->picked = at1 ? before + v0 : before;
    }
    __syncthreads();
    const int bin = s->pickBin[0], inBin = s->pickBin[1];
    rest = want - s->picked;
    // the bin's own entries; entries of one value share a bin
    float a = INFINITY, b = -INFINITY;
#pragma unroll 4
    for (unsigned int i = 0; i < count; ++i) {
      const float v = column[i * SL_THREADS];
      if (v >= least && v <= most && (bin < 0 || binOf(v) == bin)) {
        a = fminf(a, v);
        b = fmaxf(b, v);
        if (inBin <= 32) s->few[min(atomicAdd(&s->fewN, 1u), 31u)] = v;
      }
    }
    if (inBin <= 32) { // one lane per entry: what lies in front of it, by value
      __syncthreads();
      if (warp == 0) {
        const bool live = lane < inBin;
        const float v = live ? s->few[lane] : -INFINITY;
        const unsigned long long each = byMass ? units(weigh(v)) : 1ull;
        unsigned long long inFront = 0;
        unsigned int equal = 0;
#pragma unroll 1
        for (int i = 0; i < inBin; ++i) {
          const float o = __shfl_sync(0xffffffffu, v, i);
          const unsigned long long oe = __shfl_sync(0xffffffffu, each, i);
          inFront += o > v ? oe : 0ull;
          equal += o == v;
        }
        // the smallest value with less than `rest` in front of it is the border (rest >= 1: the largest qualifies)
        const bool in = live && inFront < rest;
        const float border = slWarpMin(in ? v : INFINITY);
        if (in && v == border) { // lanes of one value write the same
          s->border = border;
          s->rest = rest - inFront;
          s->equal = equal;
        }
      }
      settled = true;
    } else {
      slSpan(s, a, b);
      least = a;
      most = b;
      if (!(a < b) || bin < 0) { // one value (or, without any weight, the largest one)
        unsigned int equal = 0, allEqual;
#pragma unroll 4
        for (unsigned int i = 0; i < count; ++i) equal += column[i * SL_THREADS] == b;
        slScan<unsigned int>(equal, s->cRed[0], allEqual);
        if (threadIdx.x == 0) {
          s->border = b;
          s->rest = rest;
          s->equal = allEqual;
        }
        settled = true;
      }
    }
    __syncthreads();
  }
  const float border = s->border;
  const unsigned long long each = units(weigh(border)), per = byMass ? each : 1ull, equal = s->equal;
  unsigned long long keep = per ? (s->rest + per - 1) / per : equal, above = 0, through;
  keep = keep < 1 ? 1 : (keep > equal ? equal : keep); // a rounded limit may ask for more than there are
  if (weights) {
    forList(true, [&](float v, double w) { above += v > border ? units(w) : 0ull; });
    slScan<unsigned long long>(above, s->uRed[0], through);
    if (threadIdx.x == 0) s->through = static_cast<double>(through + keep * each) * __hiloint2double((1023 - shift) << 20, 0);
  }
  if (threadIdx.x == 0) s->ties = static_cast<unsigned int>(keep);
  __syncthreads();
}

// The next interval for a border inside [below, above): where, by the sample, `want` of the bracket's `have` entries
// (byMass: of its weight) lie above; have <= 0: not known, the sample's estimate is taken.  `open`: the interval reaches
// up to the bracket's end and down to some SL_FIRST entries.  Leaves s->lo, s->hi and (s->high) where an open one would
// begin; lo >= hi: the sample has nothing in the bracket.  Nothing here decides a result, only how soon it is found: f32
// throughout.
__device__ __forceinline__ void slChoose(SampleSmem *s, float c, float below, float above, float least, float top, bool byMass, bool open, float want,
                                         float have, int n, int samples) {
#pragma unroll 1
  for (int i = threadIdx.x; i < SL_BINS; i += SL_THREADS) s->count[i] = 0;
  __syncthreads();
  const float a = fmaxf(below, least), b = fminf(above, top); // where samples can be
  if (!(a < b) || !(b - a < INFINITY)) { // one value only, or too far apart for bins
    if (threadIdx.x == 0) s->lo = s->hi = a;
    __syncthreads();
    return;
  }
  const float step = (SL_BINS - 1) / (b - a), width = (b - a) / (SL_BINS - 1);
#pragma unroll 4
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
  const float n0 = slScan<float>(c0 + c1, s->fRed[0], cAll) + c0, n1 = n0 + c1; // entries down to either bin
  float m0 = n0, m1 = n1, q0 = n0, q1 = n1;
  mAll = qAll = cAll;
  if (byMass) {
    m0 = slScan<float>(c0 * w0 + c1 * w1, s->fRed[1], mAll) + c0 * w0;
    m1 = m0 + c1 * w1;
    q0 = slScan<float>(c0 * w0 * w0 + c1 * w1 * w1, s->fRed[0], qAll) + c0 * w0 * w0;
    q1 = q0 + c1 * w1 * w1;
  }
  const float perSample = static_cast<float>(n) / samples;
  if (cAll * perSample <= 0.6f * SL_LIST) { // the whole bracket will fit
    if (threadIdx.x == 0) {
      s->lo = below;
      s->hi = above;
    }
    __syncthreads();
    return;
  }
  const float enough = SL_FIRST / perSample;
  const bool at0 = n0 >= enough && n0 - c0 < enough, at1 = n1 >= enough && n0 < enough;
  if (at0 || at1) { // the first bin down to which there are enough: one thread's
    s->high = s->lo = fmaxf(below, a + ((at0 ? b0 : b1) - 0.5f) * width);
    s->hi = above;
  }
  if (open) {
    __syncthreads();
    return;
  }
  const float target = fminf(fmaxf(want / (have > 0.0f ? have : cAll * perSample), 0.0f), 1.0f);
  // Four standard deviations of the sampled share on both sides.  When that would not fit, fewer, which fit with a good
  // chance of a hit; or, should even two be too many, all four, whose counts then bracket the border closely.
  const float perMass = 1.0f / mAll;
  float margin = 4.0f, pad = 1.5f / samples;
  for (int round = 0;; ++round) {
    if (threadIdx.x == 0) {
      s->pickBin[0] = -1;
      s->pickBin[1] = SL_BINS;
    }
    __syncthreads();
    auto spread = [&](float q) {
      return margin * __fsqrt_rn(q * (1.0f - target) * (1.0f - target) + fmaxf(qAll - q, 0.0f) * target * target) * perMass + pad;
    };
    const float f0 = m0 * perMass, f1 = m1 * perMass, d0 = spread(q0), d1 = spread(q1);
    // highest bin that surely lies at or below the border, lowest bin that surely lies in front of it
    const int under = f0 >= target + d0 ? b0 : (f1 >= target + d1 ? b1 : -1);
    const int over = f1 <= target - d1 ? b1 : (f0 <= target - d0 ? b0 : SL_BINS);
    const int wl = __reduce_max_sync(0xffffffffu, under), wm = __reduce_min_sync(0xffffffffu, over);
    if ((threadIdx.x & 31) == 0) {
      if (wl >= 0) atomicMax(&s->pickBin[0], wl);
      if (wm < SL_BINS) atomicMin(&s->pickBin[1], wm);
    }
    __syncthreads();
    const int pLo = s->pickBin[0], pHi = s->pickBin[1];
    // how many the interval would hold, and how many with everything above it (two 16-bit counts)
    unsigned int inside = 0, both;
    if (b0 >= pLo) inside += s->count[b0] * (b0 < pHi ? 0x10001u : 0x10000u);
    if (b1 >= pLo) inside += s->count[b1] * (b1 < pHi ? 0x10001u : 0x10000u);
    slScan<unsigned int>(inside, s->cRed[0], both);
    const unsigned int sum = both & 0xffffu;
    const bool up = (both >> 16) * perSample <= 0.6f * SL_LIST; // the sample says little about a few heavy entries
    if (sum * perSample <= SL_LIST || pHi - pLo <= 1 || round == 3) {
      // bin edges lie half a bin below the bins' middles; open ends reach to the bracket's
      if (threadIdx.x == 0) {
        s->lo = pLo < 0 ? below : fmaxf(below, a + (pLo - 0.5f) * width);
        s->hi = up || pHi >= SL_BINS ? above : fminf(above, a + (pHi - 0.5f) * width);
      }
      __syncthreads();
      return;
    }
    margin = round < 2 ? margin - 1.0f : 4.0f;
  }
}

// The draw among the entries above `border` and the first `ties` equal to it, none of them below `low`.  The row is
// weighed by the 16 runs of slPass, the run that holds u times the total by 16 runs again, until there is a thread for
// each entry that is left.  The last pass may have left what is needed of the runs: KNOWN_LIST, this thread's `count` entries (all that
// stay below hi) and s->runAbove (times `scale`); KNOWN_TOP, s->runTop (the first of the largest logits is drawn).
// False: a logit lies too far above the reference.
template <typename T>
__device__ __forceinline__ bool slPick(const T *x, int n, SampleSmem *s, const Weigher &weigh, float border, unsigned int ties, float low, double u, bool exactTop,
                                       int known, unsigned int count, double scale, int32_t *out, float *prob) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // counts: above the border, and no lighter than `low` (border +inf: nothing does, a NaN compares false)
  const float above = border < INFINITY ? fmaxf(nextafterf(border, INFINITY), low) : NAN;
  const double wEqual = border >= low ? (border < INFINITY ? weigh(border) : 1.0) : 0.0;
  double sum = 0.0;
  auto weighUp = [&](const auto &v) { // a few entries
    constexpr int N = sizeof(v) / sizeof(float), SIDE = N < SL_SIDE ? N : SL_SIDE;
#pragma unroll
    for (int i0 = 0; i0 < N; i0 += SIDE) {
      bool some = false; // mostly none, when the border is high
#pragma unroll
      for (int k = 0; k < SIDE; ++k) some |= v[i0 + k] >= above;
      if (!some) continue;
      double w[SIDE];
      weigh.template each<SIDE>(v + i0, w);
#pragma unroll
      for (int k = 0; k < SIDE; ++k) {
        if (v[i0 + k] >= above) sum += w[k];
      }
    }
  };
  int from = 0, to = n;
  for (bool whole = true; whole || to - from > SL_THREADS; whole = false) {
    const int part = (to - from + SL_WARPS - 1) / SL_WARPS;
    unsigned int equal = 0;
    float big = -INFINITY; // largest logit, while it is not known
    sum = 0.0;
    if (!whole) {
      const int lo = min(to, from + warp * part), hi = min(to, lo + part);
#pragma unroll 1
      for (int i0 = lo + lane; i0 < hi; i0 += 32 * 16) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i0 + 32 * i < hi ? toF32(x[i0 + 32 * i]) : NAN;
        weighUp(v);
#pragma unroll
        for (int i = 0; i < 16; ++i) equal += v[i] == border;
      }
    } else if (known == KNOWN_LIST) { // at most SL_KEEP of them
#pragma unroll 1
      for (unsigned int i = 0; i < count; i += SL_SIDE) {
        float v[SL_SIDE];
#pragma unroll
        for (int k = 0; k < SL_SIDE; ++k) v[k] = i + k < count ? s->list[i + k][threadIdx.x] : NAN;
        weighUp(v);
#pragma unroll
        for (int k = 0; k < SL_SIDE; ++k) equal += v[k] == border;
      }
    } else if (known == KNOWN_TOP) {
      equal = lane == 0 && s->runTop[warp] == border;
    } else {
      slForRange<4>(x, s, slRun(n, warp), slRun(n, warp + 1), [&](auto &v) {
        constexpr int N = sizeof(v) / sizeof(float);
        weighUp(v);
        if (ties) {
#pragma unroll
          for (int i = 0; i < N; ++i) equal += v[i] == border;
        }
        if (!exactTop) {
#pragma unroll
          for (int i = 0; i < N; i += 2) big = slMax3(big, v[i], v[i + 1]);
        }
      });
      if (!exactTop) big = slWarpMax(big);
    }
    sum = slWarpSum(sum);
    equal = slWarpSum(equal);
    if (lane == 0) {
      s->fRed[0][warp] = big;
      s->dRed[0][warp] = whole && known == KNOWN_LIST ? sum + s->runAbove[warp] * scale : sum;
      s->cRed[0][warp] = equal;
    }
    __syncthreads();
    if (warp == 0) { // lane w: run w
      const bool mine = lane < SL_WARPS;
      const unsigned int eq = mine ? s->cRed[0][lane] : 0u, seen = slWarpScan(eq) - eq + (whole ? 0u : s->equalBefore);
      const unsigned int stay = seen < ties ? min(eq, ties - seen) : 0u;
      const double m = mine ? s->dRed[0][lane] + wEqual * stay : 0.0;
      const double run = slWarpScan(m);
      const double total = __shfl_sync(0xffffffffu, run, 31), target = whole ? u * total : s->target;
      const unsigned int hit = __ballot_sync(0xffffffffu, m > 0.0 && run > target), any = __ballot_sync(0xffffffffu, m > 0.0);
      const float largest = slWarpMax(mine ? s->fRed[0][lane] : -INFINITY);
      // none: u = 1, or the last bit of a sum taken in another order: the last run that weighs anything
      const int at = hit ? __ffs(hit) - 1 : (any ? 31 - __clz(any) : SL_WARPS - 1);
      if (lane == at) {
        s->target = target - (run - m);
        s->equalBefore = seen;
        const int lo = whole ? slRun(n, lane) : min(to, from + lane * part);
        s->from = lo;
        s->to = whole ? slRun(n, lane + 1) : min(to, lo + part);
        if (whole) {
          s->total = total;
          s->ok = exactTop || (static_cast<double>(largest) - weigh.ref) * weigh.c < SL_RISE;
        }
      }
    }
    __syncthreads();
    if (!s->ok) return false;
    from = s->from;
    to = s->to;
    __syncthreads();
  }
  // a thread per entry
  if (threadIdx.x == 0) {
    s->pickBin[0] = SL_THREADS;
    s->pickBin[1] = -1;
  }
  const int i = from + static_cast<int>(threadIdx.x);
  const float v[1] = {i < to ? toF32(x[i]) : NAN};
  sum = 0.0;
  weighUp(v);
  const bool same = v[0] == border;
  unsigned int allSame;
  double all;
  const unsigned int rank = s->equalBefore + slScan<unsigned int>(same, s->cRed[0], allSame);
  const double mine = same ? (rank < ties ? wEqual : 0.0) : sum, before = slScan<double>(mine, s->dRed[0], all);
  if (mine > 0.0) {
    if (before + mine > s->target) atomicMin(&s->pickBin[0], static_cast<int>(threadIdx.x));
    atomicMax(&s->pickBin[1], static_cast<int>(threadIdx.x));
  }
  __syncthreads();
  const int at = s->pickBin[0] < SL_THREADS ? s->pickBin[0] : max(s->pickBin[1], 0);
  if (static_cast<int>(threadIdx.x) == at) {
    *out = s->pickBin[1] >= 0 ? i : -1;
    if (prob) *prob = s->pickBin[1] >= 0 ? static_cast<float>(mine / s->total) : 0.0f;
  }
  return true;
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
  const bool greedy = !(heat > 0.0f); // the first of the largest logits: only it is a candidate
  const int32_t k = topK ? topK[row] : 0;
  const float p = topP ? topP[row] : 1.0f;
  const bool cutK = !greedy && k > 0 && k < n, cutP = !greedy && p > 0.0f && p < 1.0f;
  const float share = !greedy && minP && minP[row] > 0.0f && minP[row] <= 1.0f ? minP[row] : 0.0f;
  const double u = fmin(fmax(static_cast<double>(uniform[row]), 0.0), 1.0); // NaN: 0

  // ---- a sample: evenly spaced, or all of a short row
  const int samples = min(n, SL_SAMPLE);
  float sTop = -INFINITY, sLeast = INFINITY; // of the finite ones
  auto take = [&](int at, float v) {
    v = fmaxf(v, -INFINITY);
    s->sample[at] = v;
    sTop = fmaxf(sTop, v);
    if (v > -INFINITY) sLeast = fminf(sLeast, v);
  };
  if (n >= 4 * SL_SAMPLE) { // 16-byte vectors: a single entry costs the memory a whole sector (40 thousand clocks, not 12)
    constexpr int VEC = 16 / sizeof(T), SPOTS = SL_SAMPLE / VEC;
    const int a = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T));
    const int apart = (n - a) / VEC / SPOTS;
    uint4 raw[SPOTS / SL_THREADS];
#pragma unroll
    for (int i = 0; i < SPOTS / SL_THREADS; ++i) raw[i] = __ldg(reinterpret_cast<const uint4 *>(x + a) + (tid + i * SL_THREADS) * apart);
#pragma unroll
    for (int i = 0; i < SPOTS / SL_THREADS; ++i) {
      const T *e = reinterpret_cast<const T *>(&raw[i]);
#pragma unroll
      for (int k2 = 0; k2 < VEC; ++k2) take((i * VEC + k2) * SL_THREADS + tid, toF32(e[k2]));
    }
  } else {
    const float stride = static_cast<float>(n) / samples;
#pragma unroll 1
    for (int e = tid; e < samples; e += SL_THREADS) take(e, toF32(x[min(n - 1, static_cast<int>(e * stride))]));
  }
  __syncthreads();
  slSpan(s, sLeast, sTop);

  // What stays: entries above `border`, and of those equal to it the first `ties` by index.
  float border = -INFINITY;
  unsigned int ties = 0;
  const bool cut = cutK || cutP;
  // Without cuts and a min-p the draw needs no search: weights relative to the sample's largest logit will do, unless
  // that is so small that they overflow.
  bool exactTop = false, search = cut || greedy || share > 0.0f || !(sTop > -INFINITY && sTop < INFINITY);
  weigh.refer(sTop, greedy ? 1.0f : heat);
  for (;;) {
    int known = KNOWN_NOTHING;
    unsigned int listed = 0; // entries this thread collected in the last pass
    double scale = 1.0;      // of that pass's weights to the present reference
    float listEnd = INFINITY;
    if (search) {
      // The list holds the entries in [lo, hi); the border of the cut at work lies in [below, above).
      bool first = true, again = false, byMass = false, infinite = false, up = false;
      bool ask = cut && n > SL_SHORT && sTop > -INFINITY && sTop < INFINITY; // choose an interval first
      float below = fmaxf(fmaxf(sTop - SL_FLOOR / weigh.octaves(), -FLT_MAX), sLeast), above = INFINITY, floor = below, top = sTop;
      float lo = cut ? -FLT_MAX : INFINITY, hi = INFINITY, want = static_cast<float>(k), have = 0.0f, borderK = -INFINITY;
      float firstLo = INFINITY, firstHi = INFINITY, high = INFINITY; // where the first pass knows the weight above
      unsigned int tiesK = 0xffffffffu;
      double firstMass = 0.0, firstHiMass = 0.0, highMass = 0.0;
      double total = 0.0, atBelow = 0.0, atAbove = 0.0, limit = 0.0, mLo = 0.0, mHi = 0.0;
      int which = cutK ? 0 : 1, round = 0;
      for (bool done = false; !done;) {
        if (ask) {
          // The first interval is open unless top-k is too deep for that (256 rows of 128000, top-k 40000: 195 us with an open one, 178 closed;
          // mixed settings 300 and 239).
          slChoose(s, weigh.octaves(), below, above, sLeast, top, byMass, first ? !cutK || want <= 0.6f * SL_FIRST : up, want, have, n, samples);
          float nLo = s->lo, nHi = s->hi;
          if (first) {
            nLo = fminf(nLo, sTop);
            if (!(nLo < nHi)) nHi = INFINITY;
            if (nHi < INFINITY) high = fmaxf(s->high, nHi);
          } else if (!(nLo < nHi) || (nLo == lo && nHi == hi) || round >= 10) {
            // no help from the sample, or just what did not fit: halve the bracket in the order of the floats
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
        if (!first || infinite) listed = slPass<false, false, true>(x, n, s, weigh, lo, hi, INFINITY);
        else if (hi < INFINITY) listed = slPass<true, false, true>(x, n, s, weigh, lo, hi, high);
        else if (cutP) listed = slPass<true, true, true>(x, n, s, weigh, lo, hi, INFINITY);
        else listed = slPass<true, true, false>(x, n, s, weigh, lo, hi, INFINITY);
        const PassResult cur = s->pass;
        if (infinite) { // only the infinite ones weigh anything: both cuts count them
          border = INFINITY;
          ties = cur.cHi;
          if (cutK && static_cast<unsigned int>(k) < ties) ties = static_cast<unsigned int>(k);
          if (cutP) ties = static_cast<unsigned int>(ceil(static_cast<double>(p) * static_cast<double>(ties)));
          break;
        }
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
          const double unit = weigh.c;
          weigh.refer(cur.top, greedy ? 1.0f : heat);
          if (greedy) {
            border = cur.top;
            ties = 1;
            known = KNOWN_TOP;
            break;
          }
          if (cur.top == INFINITY) {
            infinite = true;
            ask = false;
            lo = hi = INFINITY;
            continue;
          }
          if (!cut) break;
          // From here on weights are relative to the true largest logit; the first pass's are rescaled, or taken again
          // when its reference was so far off that they may have overflowed (or there was none).
          if (!again && (cutP || hi < INFINITY)) {
            if (!(rise < SL_RISE) || weigh.c != unit) {
              again = true;
              ask = false;
              continue;
            }
            scale = weigh(sTop);
          }
          first = false;
          top = cur.top;
          floor = fmaxf(top - SL_FLOOR / weigh.octaves(), -FLT_MAX);
          total = cur.mAll * scale;
          mHi = cur.mHi * scale;
          mLo = cur.mLo * scale;
          byMass = which == 1;
          limit = byMass ? static_cast<double>(p) * total : static_cast<double>(k);
          firstLo = lo;
          firstMass = mLo;
          firstHi = hi;
          firstHiMass = mHi;
          highMass = hi < INFINITY ? cur.mHigh * scale : 0.0;
          below = floor;
          above = nextafterf(top, INFINITY);
          atBelow = byMass ? total : 0.0; // entries: not known yet
        } else {
          mHi = cur.mHi;
          mLo = cur.mLo;
          scale = 1.0;
        }
        __syncthreads(); // everyone has read the pass's result
        ask = true;
        ++round;
        // As long as the list answers: the cut's border, then the next cut.
        while (ask && !done) {
          const double hiAt = byMass ? mHi : static_cast<double>(cur.cHi), loAt = byMass ? mLo : static_cast<double>(cur.cLo);
          bool found = false;
          known = KNOWN_NOTHING;
          up = false;
          if (limit > hiAt && limit <= loAt) {
            if (cur.fits) {
              slSelect(s, weigh, listed, byMass, cutP, limit - hiAt, lo, fminf(hi, top));
              border = s->border;
              ties = s->ties;
              known = KNOWN_LIST;
              total = mHi + s->through;
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
                const double w = weigh(below), each = byMass ? fmax(w, 1e-300) : 1.0;
                const double keep = fmin(fmax(ceil((limit - hiAt) / each), 1.0), static_cast<double>(cur.cLo - cur.cHi));
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
            up = byMass; // a few heavy entries, of which the sample says little
          }
          if (!found && (above <= below || round >= 100)) { // sums that differ in their last bits left nothing between: here it is
            border = below;
            ties = 0xffffffffu;
            found = true;
          }
          if (!found) break; // another interval
          if (which == 1 && border == borderK) ties = min(ties, tiesK); // rounding must not bring back what top-k dropped
          if (which == 1 || !cutP) {
            done = true;
          } else { // top-p next, among what top-k left
            which = 1;
            borderK = border;
            tiesK = ties;
            byMass = true;
            limit = static_cast<double>(p) * total;
            below = fmaxf(border, floor);
            above = nextafterf(top, INFINITY);
            atBelow = total;
            atAbove = 0.0;
            round = 0;
            up = false;
            if (limit > firstMass) { // what the first pass knows
              above = fminf(above, firstLo);
              atAbove = firstMass;
            } else if (limit > firstHiMass) {
              if (firstHi < above) {
                above = firstHi;
                atAbove = firstHiMass;
              }
              if (firstLo > below) {
                below = firstLo;
                atBelow = firstMass;
              }
            } else {
              if (firstHi > below) {
                below = firstHi;
                atBelow = firstHiMass;
              }
              if (limit > highMass) { // the heaviest entries, of which the sample says little, are out of the way
                above = fminf(above, high);
                atAbove = highMass;
              } else if (high > below) {
                below = high;
                atBelow = highMass;
              }
            }
          }
        }
        want = static_cast<float>(limit - atAbove);
        have = atBelow > 0.0 ? fmaxf(static_cast<float>(atBelow - atAbove), 1e-30f) : 0.0f;
      }
      if (cut && border < floor) {
        border = floor;
        ties = 0xffffffffu;
        known = KNOWN_NOTHING;
      }
      listEnd = hi;
    }
    const float low = share > 0.0f ? weigh.reaches(share) : fmaxf(static_cast<float>(weigh.ref - static_cast<double>(SL_FLOOR) / weigh.c), -FLT_MAX);
    if (known == KNOWN_LIST && listEnd < low) known = KNOWN_NOTHING; // what lies above the list must stay as a whole
    if (slPick(x, n, s, weigh, border, ties, low, u, exactTop, known, listed, scale, out, prob) || exactTop) return;
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
  const size_t es = dtypeSize(dtype);
  TTB_CHECK((es == 0 || alignedTo(es, logits)) && alignedTo(4, uniform, temperature, top_k, top_p, min_p, out, prob),
            "tensors must be aligned to their elements");
  (void)workspace;
  (void)workspace_bytes;
  cudaStream_t st = asStream(stream);
  ProfScope prof("sample_logits", 4.0 * double(rows) * vocab, double(rows) * vocab * es, st);
  TTB_DISPATCH_FLOAT(dtype, T, return launchSample<T>(logits, uniform, temperature, top_k, top_p, min_p, out, prob, rows, vocab, row_stride, st))
  return TTB_OK;
}

} // extern "C"
