// What the attention of a few rows over a cache hands to its tensor-core kernel (attention_cached_tcgen05.cuh).
#pragma once

#include "common.cuh"

namespace ttb {

struct AcParams { // pointers and sizes as in ttb_sdpa_tree; window and sinks already 32-bit; `splits` runs of slots per row tile
  const int32_t *table, *lens, *parents, *draftLen;
  int *bad;
  int pages, blockSize, blocks, parentsUsers;
  int nq, heads, kvHeads, G, keys, window, sinks, splits, fmt;
  int boxes; // set by the launcher: the cache has tensor maps
  float scaleLog2;
  float *pm, *pl, *po;
};

int sdpaCachedTcgen05(const void *q, const void *k, const void *v, const void *kd, const void *vd, void *out, int dtype, int dim, int batch, const AcParams &p,
                      cudaStream_t st);

} // namespace ttb
