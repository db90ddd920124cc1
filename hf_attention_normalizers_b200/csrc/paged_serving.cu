// Paged serving on CUDA cores: appending a chunk's K/V rows to the pages,
// evicting the least attended keys, and the general (any dtype, head dim and
// page size) form of the key-weight accumulation.
#include "common.cuh"
#include "params.cuh"
#include "paged_serving.cuh"
#include "paged_walk.cuh"

namespace hfan {
namespace {

// ---------------------------------------------------------------------------
// append: the chunk of sequence b holds its last n positions, so packed row
// q_start + i goes to logical position k_len - n + i.  A thread moves one
// vector U of a K row and the same one of the V row; the grid's y axis walks
// the sequences, so that a thread finds its row without a search.  Bound by
// memory: 8 x 2048 tokens of 8 heads of 128 (134 MB): 26 us, 5.1 TB/s.
// ---------------------------------------------------------------------------
template <typename U>
__global__ void __launch_bounds__(256) append_kernel(AttnParams p, const U* k, const U* v, U* kc, U* vc,
                                                     int units, float* kw, int64_t ldw) {
  tc::allow_dependents();
  tc::wait_for_predecessor();
  const int b = blockIdx.y;
  const Geometry g = geometry(p, b);
  const int64_t row_units = (int64_t)p.hkv * units, n = g.q_len * row_units;
  for (int64_t x = blockIdx.x * 256ll + threadIdx.x; x < n; x += gridDim.x * 256ll) {
    const int i = (int)(x / row_units), r = (int)(x - i * row_units), h = r / units, c = r - h * units;
    const int pos = g.shift + i;
    if (pos < 0) {  // more new tokens than keys
      if (p.dev_status) atomicCAS(p.dev_status, kDevOk, kDevBadLength);
      continue;
    }
    const int64_t tok = key_token(p, g, b, pos);
    if (tok < 0) continue;
    const int64_t src = g.q_start + i;
    const U a = k[src * p.q_st + h * p.q_sh + c], e = v[src * p.o_st + h * p.o_sh + c];
    kc[tok * p.k_st + h * p.k_sh + c] = a;
    vc[tok * p.v_st + h * p.v_sh + c] = e;
    if (kw != nullptr && c == 0) kw[h * ldw + tok] = 0.f;
  }
}

// Cache rows of a sequence's positions; `shift`: log2 of the page size, or -1.
struct Rows {
  const int* table;
  int page_size, shift;
  int64_t tokens;
  int* status;
  __device__ __forceinline__ int operator()(int pos) const {
    const int page = table[shift >= 0 ? pos >> shift : pos / page_size];
    const int64_t row = (int64_t)page * page_size + (shift >= 0 ? pos & (page_size - 1) : pos % page_size);
    if (page < 0 || row >= tokens) {
      if (status) atomicCAS(status, kDevOk, kDevBadPage);
      return -1;
    }
    return (int)row;
  }
};

// ---------------------------------------------------------------------------
// evict, selection: one CTA per (sequence, KV head).  The weights of the
// positions before the `recent` last ones are ranked by a radix selection on
// their order-preserving integer images (11 + 11 + 10 bits, most significant
// first: a histogram finds the digit that the last kept weight has, and only
// equal prefixes count in the next pass).  Ties go to the lowest position:
// of the weights equal to the threshold the first `need` stay.  The kept
// positions are written in increasing order, each warp owning a contiguous
// range and counting with ballots.
// ---------------------------------------------------------------------------
constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32, kBins = 2048;
constexpr int kSelCache = 45056;  // weights held in shared memory (176 KB); longer sequences re-read them

// Larger floats give larger images; NaN ranks above +inf, -0 equals +0.
__device__ __forceinline__ uint32_t rank_bits(float f) {
  if (isnan(f)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int warp_sum_int(int v) { return __reduce_add_sync(0xffffffffu, v); }

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(AttnParams p, const float* kw, int64_t ldw, int budget,
                                                                   int recent, int page_shift, int* kept, int* new_lens,
                                                                   int cache) {
  tc::allow_dependents();
  tc::wait_for_predecessor();
  extern __shared__ uint32_t img[];  // [cache] images of the weights
  __shared__ int hist[kBins];
  __shared__ int wsum[2][kSelWarps];
  __shared__ int found[2];
  const int h = blockIdx.x, b = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Rows rows{p.block_table + (int64_t)b * p.max_blocks, p.page_size, page_shift, p.num_cache_tokens, p.dev_status};
  const int L = seq_len_k(p, b);
  int* out = kept + ((int64_t)b * p.hkv + h) * budget;
  if (h == 0 && threadIdx.x == 0) new_lens[b] = min(L, budget);
  if (L <= budget) {
    for (int i = threadIdx.x; i < budget; i += kSelThreads) out[i] = i < L ? i : -1;
    return;
  }
  const int late = min(recent, budget), cand = L - late, want = budget - late;  // want < cand
  const float* w = kw + (int64_t)h * ldw;
  auto fetch = [&](int j) -> uint32_t {
    const int tok = rows(j);
    return tok < 0 ? 0u : rank_bits(w[tok]);
  };
  const int held = min(cand, cache);
#pragma unroll 4
  for (int j = threadIdx.x; j < held; j += kSelThreads) img[j] = fetch(j);
  auto image = [&](int j) -> uint32_t { return j < held ? img[j] : fetch(j); };

  uint32_t prefix = 0u, mask = 0u;  // decided high bits of the threshold
  int need = want;                  // kept weights among those that match the prefix
  if (want > 0) {
    const int shifts[3] = {21, 10, 0}, widths[3] = {11, 11, 10};
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int sh = shifts[pass];
      const uint32_t dm = (1u << widths[pass]) - 1u;
      for (int i = threadIdx.x; i < kBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int j = threadIdx.x; j < cand; j += kSelThreads) {
        const uint32_t u = image(j);
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> sh) & dm], 1);
      }
      __syncthreads();
      // thread t holds bins 2 t' and 2 t' + 1 counted from the top: the
      // exclusive prefix over threads finds the bin that reaches `need`
      const int top = kBins - 1 - 2 * (int)threadIdx.x;
      const int c0 = hist[top], c1 = hist[top - 1], own = c0 + c1;
      int inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      if (lane == 31) wsum[0][warp] = inc;
      __syncthreads();
      const int before = warp_sum_int(lane < warp ? wsum[0][lane] : 0) + inc - own;
      if (before < need && before + own >= need) {
        const bool first = before + c0 >= need;
        found[0] = first ? top : top - 1;
        found[1] = need - (first ? before : before + c0);
      }
      __syncthreads();
      prefix |= (uint32_t)found[0] << sh;
      mask |= dm << sh;
      need = found[1];
    }
  }
  __syncthreads();

  // Warp w owns positions [w seg, (w + 1) seg), seg a multiple of 32.
  const int seg = ((cand + kSelThreads - 1) / kSelThreads) * 32;
  const int lo = min(warp * seg, cand), hi = min(lo + seg, cand);
  int gt = 0, eq = 0;
  if (want > 0) {
    for (int j0 = lo; j0 < hi; j0 += 32) {
      const int j = j0 + lane;
      const uint32_t u = j < hi ? image(j) : 0u;
      gt += __popc(__ballot_sync(0xffffffffu, j < hi && u > prefix));
      eq += __popc(__ballot_sync(0xffffffffu, j < hi && u == prefix));
    }
  }
  if (lane == 0) {
    wsum[0][warp] = gt;
    wsum[1][warp] = eq;
  }
  __syncthreads();
  int at = warp_sum_int(lane < warp ? wsum[0][lane] : 0);
  int ties = warp_sum_int(lane < warp ? wsum[1][lane] : 0);
  at += min(ties, need);
  if (want > 0) {
    for (int j0 = lo; j0 < hi; j0 += 32) {
      const int j = j0 + lane;
      const uint32_t u = j < hi ? image(j) : 0u;
      const unsigned below = (1u << lane) - 1u;
      const unsigned be = __ballot_sync(0xffffffffu, j < hi && u == prefix);
      const bool keep = j < hi && (u > prefix || (u == prefix && ties + __popc(be & below) < need));
      const unsigned bk = __ballot_sync(0xffffffffu, keep);
      if (keep) out[at + __popc(bk & below)] = j;
      at += __popc(bk);
      ties += __popc(be);
    }
  }
  for (int i = threadIdx.x; i < late; i += kSelThreads) out[want + i] = cand + i;
}

// ---------------------------------------------------------------------------
// evict, move: kept position kept[i] >= i goes to logical position i.  One CTA
// owns a strip (some columns of K, of V, or the weights) of one (sequence, KV
// head), so strips are independent; within a strip the rows go in steps, in
// increasing order.  A step reads rows kept[i] >= i of its own i range, so only
// its own writes can hit its reads: one barrier between the loads and the
// stores of a step, and the loads of the next one (rows beyond every row
// written so far) are in flight before them.
//
// Bound by memory: each kept row is read and written once.  Strips are whole
// rows when there are enough (sequence, head) pairs to fill the SMs; else they
// get narrower, down to a 32-byte sector, since a strip goes at the pace of one
// load after the other.  32 sequences of 16k keys cut to 4k (1.07 GB): 265 us,
// 4.0 TB/s -- the 256-byte rows lie scattered over the pages; more rows in
// flight per thread were slower (four: 300 us, eight: 440), 256 threads too
// (380), and narrow strips no faster (270).
// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 512;

template <typename U>
__device__ void move_strip(const Rows& rows, const int* kept, int count, U* base, int64_t st, int width, int lanes) {
  const int step = kMoveThreads / lanes, c = threadIdx.x % lanes, r0 = threadIdx.x / lanes;
  const bool on = r0 < step && c < width;
  auto load = [&](int i, U& v) -> int {  // the row that v goes to, or -1
    if (!on || i >= count) return -1;
    const int j = kept[i];
    if (j == i) return -1;
    const int src = rows(j);
    if (src < 0) return -1;
    v = base[(int64_t)src * st + c];
    return rows(i);
  };
  U v0, v1;
  int d0 = load(r0, v0);
  for (int i0 = 0; i0 < count; i0 += 2 * step) {
    const int d1 = load(i0 + step + r0, v1);
    __syncthreads();
    if (d0 >= 0) base[(int64_t)d0 * st + c] = v0;
    d0 = load(i0 + 2 * step + r0, v0);
    __syncthreads();
    if (d1 >= 0) base[(int64_t)d1 * st + c] = v1;
  }
}

template <typename U>
__global__ void __launch_bounds__(kMoveThreads, 4) evict_move_kernel(AttnParams p, U* kc, U* vc, float* kw, int64_t ldw,
                                                                  int units, int slice, int slices, int budget,
                                                                  int page_shift, const int* kept) {
  tc::allow_dependents();
  tc::wait_for_predecessor();
  const int h = blockIdx.y, b = blockIdx.z;
  const int L = seq_len_k(p, b);
  if (L <= budget) return;
  const int* kp = kept + ((int64_t)b * p.hkv + h) * budget;
  const Rows rows{p.block_table + (int64_t)b * p.max_blocks, p.page_size, page_shift, p.num_cache_tokens, p.dev_status};
  const int s = blockIdx.x;
  if (s == 2 * slices) {
    move_strip<float>(rows, kp, budget, kw + (int64_t)h * ldw, 1, 1, 1);
  } else {
    const int c0 = (s % slices) * slice, width = min(slice, units - c0);
    if (s < slices)
      move_strip<U>(rows, kp, budget, kc + (int64_t)h * p.k_sh + c0, p.k_st, width, slice);
    else
      move_strip<U>(rows, kp, budget, vc + (int64_t)h * p.v_sh + c0, p.v_st, width, slice);
  }
}

// ---------------------------------------------------------------------------
// key weights, general form: one warp per key, lanes over the packed (token,
// head) rows of the KV group; fp32 dot products.
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) key_weights_kernel(AttnParams p, float* kw, int64_t ldw) {
  extern __shared__ float ks[];  // [8][D]
  const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Geometry g = geometry(p, b);
  const int j = blockIdx.x * 8 + warp;
  if (j >= g.k_len) return;
  const int64_t tok = key_token(p, g, b, j);
  if (tok < 0) return;
  const T* kr = static_cast<const T*>(p.k) + tok * p.k_st + kvh * p.k_sh;
  float* kf = ks + warp * p.d;
  for (int d = lane; d < p.d; d += 32) kf[d] = to_f32<T>(kr[d]);
  __syncwarp();
  const int G = p.hq / p.hkv;
  const float zs = p.norm == HFAN_SOFTMAX1 ? p.scale * kLog2e : (p.norm == HFAN_SPARSEMAX ? p.scale : 0.5f * p.scale);
  const int i0 = p.causal ? max(0, j - g.shift) : 0;
  float acc = 0.f;
  for (int64_t r = (int64_t)i0 * G + lane; r < (int64_t)g.q_len * G; r += 32) {
    const int i = (int)(r / G), h = kvh * G + (int)(r - (int64_t)i * G);
    const T* qr = static_cast<const T*>(p.q) + (int64_t)(g.q_start + i) * p.q_st + h * p.q_sh;
    float s = 0.f;
    for (int d = 0; d < p.d; ++d) s = fmaf(to_f32<T>(qr[d]), kf[d], s);
    const int64_t si = stat_index(p, g, h, i);
    const float s0 = p.stats[si];
    if (p.norm == HFAN_SOFTMAX1)
      acc += exp2f(s * zs - s0) / p.stats[(int64_t)p.hq * p.rows_total + si];
    else
      acc += sparse_prob(p.norm, s * zs, s0);
  }
  acc = warp_sum(acc);
  if (lane == 0 && acc != 0.f) atomicAdd(kw + (int64_t)kvh * ldw + tok, acc);
}

int page_shift(const AttnParams& p) { return (p.page_size & (p.page_size - 1)) == 0 ? __builtin_ctz(p.page_size) : -1; }

int elem_bytes(int dtype) { return dtype == HFAN_FLOAT32 ? 4 : 2; }

bool vec16(const void* ptr, int64_t a, int64_t b, int es) {
  return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && (a * es) % 16 == 0 && (b * es) % 16 == 0;
}

template <typename U>
cudaError_t append_t(int dtype, const AttnParams& p0, float* kw, int64_t ldw, cudaStream_t s) {
  AttnParams p = p0;
  const int per = (int)sizeof(U) / elem_bytes(dtype), units = p.d / per;
  p.q_st /= per; p.q_sh /= per; p.o_st /= per; p.o_sh /= per;
  p.k_st /= per; p.k_sh /= per; p.v_st /= per; p.v_sh /= per;
  // about four vectors a thread, and enough CTAs to fill the SMs
  const int64_t vecs = (int64_t)p.rows_total * p.hkv * units;
  int64_t gx = (vecs + (int64_t)p.batch * 1024 - 1) / ((int64_t)p.batch * 1024);
  gx = gx < 1 ? 1 : (gx > 4096 ? 4096 : gx);
  return launch_dependent(append_kernel<U>, dim3((unsigned)gx, p.batch), 256, 0, s, p, static_cast<const U*>(p.q),
                          static_cast<const U*>(p.o), static_cast<U*>(const_cast<void*>(p.k)),
                          static_cast<U*>(const_cast<void*>(p.v)), units, kw, ldw);
}

template <typename U>
cudaError_t move_t(int dtype, const AttnParams& p0, float* kw, int64_t ldw, int budget, const int* kept, cudaStream_t s) {
  AttnParams p = p0;
  const int per = (int)sizeof(U) / elem_bytes(dtype), units = p.d / per;
  p.k_st /= per; p.k_sh /= per; p.v_st /= per; p.v_sh /= per;
  // vectors of a strip's row: the whole row, halved while the strips would not
  // give every SM two CTAs, but no less than a sector
  const int sector = 32 / (int)sizeof(U);
  int slice = units < 64 ? units : 64;
  while (slice % 2 == 0 && slice / 2 >= sector && (int64_t)p.batch * p.hkv * 2 * ((units + slice - 1) / slice) < 2 * sm_count())
    slice /= 2;
  const int slices = (units + slice - 1) / slice;
  return launch_dependent(evict_move_kernel<U>, dim3(2 * slices + 1, p.hkv, p.batch), kMoveThreads, 0, s, p,
                          static_cast<U*>(const_cast<void*>(p.k)), static_cast<U*>(const_cast<void*>(p.v)), kw, ldw, units,
                          slice, slices, budget, page_shift(p), kept);
}

}  // namespace

cudaError_t serving_append(int dtype, const AttnParams& p, float* kw, int64_t ldw, cudaStream_t s) {
  const int es = elem_bytes(dtype);
  const bool v = (p.d * es) % 16 == 0 && vec16(p.q, p.q_st, p.q_sh, es) && vec16(p.o, p.o_st, p.o_sh, es) &&
                 vec16(p.k, p.k_st, p.k_sh, es) && vec16(p.v, p.v_st, p.v_sh, es);
  if (v) return append_t<uint4>(dtype, p, kw, ldw, s);
  return es == 4 ? append_t<uint32_t>(dtype, p, kw, ldw, s) : append_t<uint16_t>(dtype, p, kw, ldw, s);
}

cudaError_t serving_evict(int dtype, const AttnParams& p, float* kw, int64_t ldw, int budget, int recent, int* kept,
                          int* new_lens, cudaStream_t s) {
  const int cache = p.len_k < kSelCache ? p.len_k : kSelCache;
  const size_t smem = (size_t)cache * 4;
  // (asked for at every length: what a launch may have by default holds the static arrays too)
  cudaError_t e = allow_smem<evict_select_kernel>(kSelCache * 4);
  if (e != cudaSuccess) return e;
  e = launch_dependent(evict_select_kernel, dim3(p.hkv, p.batch), kSelThreads, smem, s, p, static_cast<const float*>(kw), ldw,
                       budget, recent, page_shift(p), kept, new_lens, cache);
  if (e != cudaSuccess || p.len_k <= budget) return e;
  const int es = elem_bytes(dtype);
  const bool v = (p.d * es) % 16 == 0 && vec16(p.k, p.k_st, p.k_sh, es) && vec16(p.v, p.v_st, p.v_sh, es);
  if (v) return move_t<uint4>(dtype, p, kw, ldw, budget, kept, s);
  return es == 4 ? move_t<uint32_t>(dtype, p, kw, ldw, budget, kept, s)
                 : move_t<uint16_t>(dtype, p, kw, ldw, budget, kept, s);
}

cudaError_t serving_key_weights(int dtype, const AttnParams& p, float* kw, int64_t ldw, cudaStream_t s) {
  const dim3 grid((unsigned)((p.len_k + 7) / 8), p.hkv, p.batch);
  const size_t smem = 8 * p.d * sizeof(float);
  if (dtype == HFAN_FLOAT32) key_weights_kernel<float><<<grid, 256, smem, s>>>(p, kw, ldw);
  else if (dtype == HFAN_FLOAT16) key_weights_kernel<__half><<<grid, 256, smem, s>>>(p, kw, ldw);
  else key_weights_kernel<__nv_bfloat16><<<grid, 256, smem, s>>>(p, kw, ldw);
  return cudaGetLastError();
}

}  // namespace hfan
