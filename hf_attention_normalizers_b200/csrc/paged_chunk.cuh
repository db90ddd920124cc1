// Shared by the tensor-core kernels of the ragged chunk attention: how packed
// query rows and key tiles are cut, and the loads of a page-table key tile.
//
// The G = Hq / Hkv query heads of a KV head read the same keys, so the rows of
// a tile are (token, head) pairs, head fastest: a tile of 128 rows holds `tpb`
// tokens (128 / G rounded down, or fewer when no sequence brings that many)
// and every byte of K and V serves the whole group.
#pragma once

#include <atomic>

#include "params.cuh"
#include "tc_common.cuh"

namespace hfan {

constexpr int kTileRows = 128;  // packed (token, head) rows of one tile
constexpr int kTileKeys = 128;

struct ChunkPlan {
  int group;     // query heads per KV head
  int tpb;       // tokens per tile
  int box_rows;  // rows of one TMA box of a page: a power of two that divides the page size, 8 .. 128
  int pairs;     // upper bound of the tile pairs of all sequences
};

// Tokens of sequence b and the first of them, clamped as geometry() does.
__device__ __forceinline__ int chunk_tokens(const AttnParams& p, int b, int* start) {
  const int s = min(max(p.cu_q[b], 0), p.rows_total);
  *start = s;
  return min(max(p.cu_q[b + 1], s), p.rows_total) - s;
}

// Records offsets that chunk_tokens clamped, as geometry() does (which nobody
// calls for a sequence that they leave empty).  For threads with nothing else to
// do: in the searches of all warps the test cost a small decode 0.5 us.
__device__ __forceinline__ void record_bad_offsets(const AttnParams& p, int thread, int threads) {
  for (int b = thread; b < p.batch; b += threads) {
    int s;
    const int n = chunk_tokens(p, b, &s);
    if ((s != p.cu_q[b] || s + n != p.cu_q[b + 1]) && p.dev_status) atomicCAS(p.dev_status, kDevOk, kDevBadLength);
  }
}

// The x-th group of `per` tokens over all sequences (the last of a sequence
// may hold fewer).  Whole-warp call, uniform result; false past the last one.
__device__ __forceinline__ bool find_group(const AttnParams& p, int per, int x, int* b, int* idx) {
  const int lane = threadIdx.x & 31;
  for (int base = 0; base < p.batch; base += 32) {
    int cnt = 0, s;
    if (base + lane < p.batch) cnt = (chunk_tokens(p, base + lane, &s) + per - 1) / per;
    int inc = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, inc > x);
    if (hit) {
      const int l = __ffs(hit) - 1;
      *b = base + l;
      *idx = x - __shfl_sync(0xffffffffu, inc - cnt, l);
      return true;
    }
    x -= __shfl_sync(0xffffffffu, inc, 31);
  }
  return false;
}

// Cache row of the first key of lane's box of key tile kt (-1: no such box).
// A page id outside the cache gives num_cache_tokens, which the tensor map
// fills with zeros, and is recorded.
__device__ __forceinline__ int tile_box_row(const AttnParams& p, const ChunkPlan& c, int b, int k_len, int kt) {
  const int off = (threadIdx.x & 31) * c.box_rows, key = kt * kTileKeys + off;
  if (off >= kTileKeys || key >= k_len) return -1;
  const int page = p.block_table[(int64_t)b * p.max_blocks + key / p.page_size];
  const int64_t row = (int64_t)page * p.page_size + key % p.page_size;
  if (page < 0 || row >= p.num_cache_tokens) {
    if (p.dev_status) atomicCAS(p.dev_status, kDevOk, kDevBadPage);
    return (int)p.num_cache_tokens;
  }
  return (int)row;
}

// Loads the boxes of one key tile (rows from tile_box_row) into a stage of
// NH swizzled halves.  Whole-warp call; rows of keys past k_len in the last
// box hold whatever the page holds, boxes past it keep the stage's old bytes.
template <int NH>
__device__ __forceinline__ void load_key_tile_tma(uint8_t* stage, const CUtensorMap* map, uint64_t* bar, int row,
                                                  int box_rows, int kvh) {
  const unsigned have = __ballot_sync(0xffffffffu, row >= 0);
  if ((threadIdx.x & 31) == 0)
    tc::mbar_arrive_expect_tx(bar, (uint32_t)__popc(have) * (uint32_t)box_rows * 128u * NH);
  __syncwarp();
  if (row >= 0) {
    uint8_t* dst = stage + (threadIdx.x & 31) * box_rows * 128;
#pragma unroll
    for (int hh = 0; hh < NH; ++hh) tc::tma_load_4d(dst + hh * tc::kHalf, map, bar, 64 * hh, row, kvh, 0);
  }
}

// ------------------------------------------------------------------ host
inline int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Lets `kernel` use `smem` bytes of dynamic shared memory: once per kernel and
// device (the attribute call costs a launch about as much as its arguments).
template <auto Kernel>
cudaError_t allow_smem(int smem) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// (dim, head, token) map of packed rows: a box is one tile, rows token-major.
inline bool make_row_map(CUtensorMap* m, const AttnParams& p, bool bf16, const ChunkPlan& c) {
  return tc::make_map_box(m, p.q, bf16, {(cuuint64_t)p.d, (cuuint64_t)p.hq, (cuuint64_t)p.rows_total, 1},
                      {p.q_sh, p.q_st, p.q_st * p.rows_total}, {64, (cuuint32_t)c.group, (cuuint32_t)c.tpb, 1});
}
inline bool make_page_map(CUtensorMap* m, const void* cache, int64_t st, int64_t sh, const AttnParams& p, bool bf16,
                   const ChunkPlan& c) {
  return tc::make_map(m, cache, bf16, p.d, p.num_cache_tokens, p.hkv, 1, st, sh, p.num_cache_tokens * st, c.box_rows);
}

// Thresholds of the sparse normalizers into p.stats, and the output of every
// unit whose flag it leaves 0 (flags [pairs][hkv]).
cudaError_t chunk_sparse_scan(int dtype, const AttnParams& p, const ChunkPlan& c, int* flags, cudaStream_t s);

// softmax1 with at most 32 packed rows a sequence (paged_few_tc.cu); adds to
// the key weights kw [hkv][ldw] when it is given.
bool chunk_few_applies(const AttnParams& p, const ChunkPlan& c, bool weights);
int64_t chunk_few_workspace(const AttnParams& p, const ChunkPlan& c, bool weights);
cudaError_t chunk_few_fwd(int dtype, const AttnParams& p, const ChunkPlan& c, float* kw, int64_t ldw, void* workspace,
                          cudaStream_t s);

}  // namespace hfan
