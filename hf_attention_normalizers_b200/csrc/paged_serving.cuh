// Host entry points of the paged serving kernels.
//
// AttnParams fields as they are used here: cu_q [batch + 1] offsets of the
// packed new tokens, rows_total their number, seq_lens / block_table /
// page_size the cache's bookkeeping, len_k an upper bound of seq_lens.
// Key weights are float32 [heads_kv][ld], one accumulator per cache slot.
#pragma once

#include "params.cuh"

namespace hfan {

// A launch that may be set up while its predecessor on the stream still runs:
// the kernel calls wait_for_predecessor (tc_ptx.cuh) before it touches memory.
// Kernels of a few microseconds follow one another here, and their prologues
// (barriers, TMEM, tensor maps) and launches hide under each other.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// q = new K rows (q_st, q_sh), o = new V rows (o_st, o_sh) -> caches k, v.
cudaError_t serving_append(int dtype, const AttnParams& p, float* kw, int64_t ldw, cudaStream_t s);
cudaError_t serving_evict(int dtype, const AttnParams& p, float* kw, int64_t ldw, int budget, int recent, int* kept,
                          int* new_lens, cudaStream_t s);
// kw[kvh][slot] += sum of p over the chunk's rows of the KV group (p.stats: what the forward saved).
cudaError_t serving_key_weights(int dtype, const AttnParams& p, float* kw, int64_t ldw, cudaStream_t s);

// Tensor-core form (paged_chunk_tc.cu) of the chunk attention and, when kw is
// given, the key weights.  The workspace size depends on sizes alone, so it may
// be asked for before the tensors are known.
bool chunk_tc_supported(int dtype, const AttnParams& p);
int64_t chunk_tc_workspace(const AttnParams& p, bool weights);
cudaError_t chunk_tc_fwd(int dtype, const AttnParams& p, float* kw, int64_t ldw, void* workspace, cudaStream_t s);

}  // namespace hfan
