// Sampling from whole rows of logits (ttb_sample_logits).  For a row x of `vocab` logits, temperature T:
//   w_i = exp((x_i - max x) / T)                        weights; NaN and -inf logits have none
//   top-k   the k largest logits stay (equal ones: the lower index first)
//   top-p   of those, in the same order, the shortest prefix whose weight reaches p of their sum
//   min-p   of those, the ones with w_i >= min_p
//   draw    the first i, in index order, at which the running sum of what stayed exceeds u times its total
// Weights are summed as 64-bit integers (units of 2^-40 of the largest weight): sums are exact whatever their order,
// so the token does not depend on how the row is split over threads, and a weight below 2^-41 counts as none.
//
// One CTA per row.  The cuts are one radix selection each over the order-preserving 32-bit image of the logits: four
// rounds of 256 bins (count and weight per bin), after which the border value is known exactly and what is left to
// decide is how many of the entries equal to it stay.
#include "common.cuh"

namespace ttb {

constexpr int SL_THREADS = 1024;
constexpr float SL_UNIT = 1099511627776.0f; // 2^40
constexpr int64_t SL_MAX_VOCAB = 1 << 22;   // 2^22 weights of 2^40 units fit 63 bits

// Order-preserving image: larger floats have larger images.  -0 is folded onto 0 first (they are equal).
__device__ __forceinline__ uint32_t slKey(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct SampleRow {
  float top;      // largest logit
  float c;        // log2(e) / T
  float cLow;     // what c lost to rounding
};

// Weight in units.  d c is split into a rounded product and its error, so that the weight's relative error stays
// near 2^-23 however far the logit is from the top.
__device__ __forceinline__ float slWeightF(float x, const SampleRow &r) {
  if (x == r.top) return 1.0f;             // also +inf against +inf
  if (!(x > -INFINITY)) return 0.0f;       // -inf, NaN
  const float d = x - r.top;
  if (!(d > -INFINITY)) return 0.0f;       // a finite logit under a +inf one
  const float hi = d * r.c, lo = fmaf(d, r.c, -hi) + d * r.cLow;
  const float w = exp2f(hi);
  return isfinite(lo) ? fmaf(w * lo, 0.6931471805599453f, w) : w;
}
__device__ __forceinline__ unsigned long long slUnits(float w) { return __float2ull_rn(w * SL_UNIT); }

template <typename V> __device__ __forceinline__ V slWarpSum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(SL_THREADS)
    sampleLogitsKernel(const T *__restrict__ logits, const float *__restrict__ uniform, const float *__restrict__ temperature,
                       const int32_t *__restrict__ topK, const float *__restrict__ topP, const float *__restrict__ minP, int32_t *__restrict__ out,
                       float *__restrict__ prob, int64_t vocab, int64_t rowStride) {
  __shared__ unsigned long long mass[256], warpMass[32];
  __shared__ unsigned int count[256];
  __shared__ unsigned long long sRest;  // what is left of the limit in front of the border
  __shared__ unsigned long long sTotal;
  __shared__ uint32_t sPrefix;
  __shared__ int sPick;
  __shared__ float warpTop[32];
  __shared__ long long warpAt[32];
  pdlLaunchDependents();
  pdlWait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const T *x = logits + row * rowStride;
  const int n = static_cast<int>(vocab);

  // ---- the largest logit and its first index
  float top = -INFINITY;
  int at = 0x7fffffff;
  for (int i = tid; i < n; i += SL_THREADS) {
    const float v = toF32(x[i]);
    if (v > top) {
      top = v;
      at = i;
    }
  }
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
    warpTop[warp] = top;
    warpAt[warp] = at;
  }
  __syncthreads();
  for (int w = 0; w < 32; ++w) {
    if (warpTop[w] > top || (warpTop[w] == top && warpAt[w] < at)) {
      top = warpTop[w];
      at = static_cast<int>(warpAt[w]);
    }
  }
  const float heat = temperature ? temperature[row] : 1.0f;
  if (top == -INFINITY || !(heat > 0.0f)) { // nothing to choose from, or greedy
    if (tid == 0) {
      out[row] = top == -INFINITY ? -1 : at;
      if (prob) prob[row] = top == -INFINITY ? 0.0f : 1.0f;
    }
    return;
  }
  SampleRow r;
  r.top = top;
  const double cd = 1.4426950408889634 / static_cast<double>(heat);
  r.c = static_cast<float>(cd);
  r.cLow = isfinite(r.c) ? static_cast<float>(cd - static_cast<double>(r.c)) : 0.0f;

  // What stays: keys above `border`, and of those equal to it the first `ties` by index; weights of at least `low`.
  uint32_t border = 0;
  unsigned long long ties = ~0ull;
  const float low = minP && minP[row] > 0.0f && minP[row] <= 1.0f ? minP[row] : 0.0f;

  // Narrows (border, ties) to the prefix, in descending order, that the limit allows: `limit` entries, or entries as
  // long as the weight in front of them is below `limit`.
  auto cut = [&](bool byMass, unsigned long long limit) {
    uint32_t prefix = 0;
    unsigned long long rest = limit;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) {
        mass[tid] = 0;
        count[tid] = 0;
      }
      __syncthreads();
      for (int i = tid; i < n; i += SL_THREADS) {
        const float v = toF32(x[i]);
        const uint32_t key = slKey(v);
        const float w = slWeightF(v, r);
        if (!(v > -INFINITY) || key < border) continue;
        if (shift < 24 && (key >> (shift + 8)) != prefix) continue;
        const int bin = (key >> shift) & 255;
        atomicAdd(&count[bin], 1u);
        if (byMass) atomicAdd(&mass[bin], slUnits(w));
      }
      __syncthreads();
      if (tid == 0) { // walk down to the bin in which the limit is used up
        int bin = 255, lastBin = -1;
        unsigned long long left = rest;
        for (; bin >= 0; --bin) {
          if (!count[bin]) continue;
          unsigned long long have = byMass ? mass[bin] : count[bin];
          // entries of the border value that an earlier cut did not keep must not count
          if (shift == 0 && ((prefix << 8) | static_cast<uint32_t>(bin)) == border && count[bin] > ties)
            have = byMass ? have / count[bin] * ties : ties;
          lastBin = bin;
          if (left <= have) break;
          left -= have;
        }
        if (bin < 0) { // the limit is not reached: the last bin that holds anything is the border
          bin = lastBin;
          left = ~0ull;
        }
        sPrefix = (prefix << 8) | static_cast<uint32_t>(bin);
        sRest = left;
        if (shift == 0) {
          unsigned long long each = byMass ? mass[bin] / count[bin] : 1;
          sTotal = left == ~0ull ? ~0ull : (each ? (left + each - 1) / each : ~0ull);
        }
      }
      __syncthreads();
      prefix = sPrefix;
      rest = sRest;
      if (rest == ~0ull) { // everything stays
        __syncthreads();
        return;
      }
    }
    const unsigned long long keep = sTotal > 0 ? sTotal : 1;
    ties = border == prefix ? min(ties, keep) : keep;
    border = prefix;
    __syncthreads();
  };
  // Every warp owns a run of indices.
  const int perWarp = ((n + 31) / 32 + 31) / 32 * 32;
  const int32_t k = topK ? topK[row] : 0;
  if (k > 0 && k < n) cut(false, static_cast<unsigned long long>(k));
  const float p = topP ? topP[row] : 1.0f;

  // Entries equal to the border: the number in front of each warp's run decides which of them stay.
  auto sumRun = [&](bool minimum, unsigned long long equalBefore, unsigned long long &equalSeen) -> unsigned long long {
    unsigned long long sum = 0;
    equalSeen = 0;
    const int lo = warp * perWarp, hi = min(n, lo + perWarp);
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      const float v = i < hi ? toF32(x[i]) : -INFINITY;
      const float w = slWeightF(v, r);
      const uint32_t key = slKey(v);
      const bool live = v > -INFINITY, equal = live && key == border;
      const unsigned int eq = __ballot_sync(0xffffffffu, equal);
      const unsigned long long rank = equalBefore + equalSeen + __popc(eq & ((1u << lane) - 1u));
      if (live && (key > border || (equal && rank < ties)) && (!minimum || w >= low)) sum += slUnits(w);
      equalSeen += __popc(eq);
    }
    return slWarpSum(sum);
  };
  __shared__ unsigned long long warpEqual[32];
  auto sums = [&](bool minimum) -> unsigned long long { // fills warpMass and warpEqual (exclusive), returns the total
    unsigned long long eq;
    sumRun(minimum, 0, eq);
    if (lane == 0) warpEqual[warp] = eq;
    __syncthreads();
    unsigned long long before = 0;
    for (int w = 0; w < warp; ++w) before += warpEqual[w];
    const unsigned long long mine = sumRun(minimum, before, eq);
    if (lane == 0) warpMass[warp] = mine;
    __syncthreads();
    if (lane == 0) warpEqual[warp] = before;
    unsigned long long total = 0;
    for (int w = 0; w < 32; ++w) total += warpMass[w];
    __syncthreads();
    return total;
  };
  if (p > 0.0f && p < 1.0f) {
    const unsigned long long total = sums(false);
    // an entry stays while the weight in front of it is below p times the total
    const unsigned long long limit = static_cast<unsigned long long>(ceil(static_cast<double>(p) * static_cast<double>(total)));
    cut(true, limit);
  }
  const unsigned long long total = sums(true);
  // first running sum above u * total, i.e. the smallest number of whole units above it
  double u = uniform ? static_cast<double>(uniform[row]) : 0.0;
  u = u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0;
  unsigned long long target = static_cast<unsigned long long>(u * static_cast<double>(total));
  if (target >= total) target = total - 1;
  if (tid == 0) sPick = -1;
  __syncthreads();
  unsigned long long before = 0;
  for (int w = 0; w < warp; ++w) before += warpMass[w];
  if (target >= before && target < before + warpMass[warp]) { // exactly one warp
    unsigned long long equalSeen = warpEqual[warp];
    const int lo = warp * perWarp, hi = min(n, lo + perWarp);
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      const float v = i < hi ? toF32(x[i]) : -INFINITY;
      const float w = slWeightF(v, r);
      const uint32_t key = slKey(v);
      const bool live = v > -INFINITY, equal = live && key == border;
      const unsigned int eq = __ballot_sync(0xffffffffu, equal);
      const unsigned long long rank = equalSeen + __popc(eq & ((1u << lane) - 1u));
      unsigned long long mine = 0;
      if (live && (key > border || (equal && rank < ties)) && w >= low) mine = slUnits(w);
      equalSeen += __popc(eq);
      unsigned long long run = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long left = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += left;
      }
      const unsigned int hit = __ballot_sync(0xffffffffu, before + run > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          out[row] = i;
          if (prob) prob[row] = static_cast<float>(static_cast<double>(mine) / static_cast<double>(total));
        }
        return;
      }
      before += __shfl_sync(0xffffffffu, run, 31);
    }
  }
}

} // namespace ttb

using namespace ttb;

extern "C" {

size_t ttb_sample_logits_workspace_bytes(int64_t rows, int64_t vocab) {
  (void)rows;
  (void)vocab;
  return 0;
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
  TTB_DISPATCH_FLOAT(dtype, T, TTB_CUDA(launchPdl(sampleLogitsKernel<T>, dim3(static_cast<unsigned>(rows)), dim3(SL_THREADS), 0, st,
                                                  static_cast<const T *>(logits), static_cast<const float *>(uniform),
                                                  static_cast<const float *>(temperature), static_cast<const int32_t *>(top_k),
                                                  static_cast<const float *>(top_p), static_cast<const float *>(min_p), static_cast<int32_t *>(out),
                                                  static_cast<float *>(prob), vocab, row_stride)))
  countLaunch();
  TTB_LAUNCH_CHECK();
  return TTB_OK;
}

} // extern "C"
