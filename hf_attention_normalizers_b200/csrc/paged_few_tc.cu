// softmax1 attention of a few new tokens per sequence (at most 32 packed
// (token, head) rows: decoding, and short speculative chunks) over a paged
// cache, and its key weights.  16-bit inputs, head_dim 64 / 128.
//
// Bound by reading K and V once, so the tensor cores run on the transposed
// problem, where the keys fill the 128 rows of an MMA and the packed rows are
// its few columns:  S^T = K Q^T  (128 keys x NC), then  O^T += V^T P^T
// (head dim x NC).  A thread owns a key: it exponentiates NC scores instead of
// the 128 that a mostly empty query tile would cost, and writes them as one
// column of P^T (the B operand) to shared memory.
//
//   warps 0-3  softmax (thread = key, then = head dim when O^T is written)
//   warp 4     producer: Q of a piece, K and V tiles through one deep ring
//   warp 5     MMA issuer; S of the next tile is issued before P V of this one
//
// The reference m of a row follows the maximum lazily and only when a score
// passes it by 2^8, which one vote of the four warps finds; a decoded row
// seldom takes that path. It starts at the implicit zero logit in bfloat16,
// whose exponents reach as far as float32's. In float16, where P below 2^-14
// loses bits and vanishes below 2^-25, a row whose first tile stays below that
// logit starts 2^8 under its maximum there, and all follow past 2^15. The CTAs
// walk equal stretches of all key tiles of the batch (paged_walk.cuh).
//
// P enters P V as two 16-bit parts, P rounded and what the rounding left, so
// that only the result is rounded (one part: output errors 1.5 times those of
// a float32 computation that rounds its result).  The tensor pipe has room: 8
// sequences of 32k keys take 191.0 us with two parts and 190.3 with one, 16
// chunks of 8 tokens on 8k keys 123.2 and 121.0 (medians of graph launches, L2
// flushed).
//
// Measured: 8 sequences of 32k keys, one token each, 8 KV heads of 128: 1.07 GB
// in 178 us, 6.0 TB/s of DRAM reads (0.92 of a copy); 4 sequences of up to 2k
// keys: 12 us, of which setting up (barriers, TMEM, the walk) takes 2 and the
// first tile's loads 2.
//
// With key weights the raw scores are kept (four bytes a row and key, against
// the 2 D bytes of the K row), so that the pass over the final statistics reads them
// instead of K.
#include <cuda.h>

#include "common.cuh"
#include "paged_serving.cuh"
#include "paged_walk.cuh"
#include "tc_ptx.cuh"

namespace hfan {
namespace {

using namespace tc;

constexpr int kFewThreads = 192;

// A row's reference moves when a score passes it by kRescale octaves.  float16:
// P stays below 2^15, and a new reference lies kHeadroom16 octaves below the
// maximum (paged_walk.cuh).
template <bool BF16>
constexpr float kRescale = BF16 ? 8.f : 15.f;

constexpr int kSumStride = 132;  // floats; rows of 128 start in different banks

template <int HD, int NC>
struct FewLayout {
  static constexpr int NH = HD / 64, NS = HD == 128 ? (NC == 16 ? 6 : 5) : (NC == 16 ? 10 : 9);
  static constexpr uint32_t TILE = NH * kHalf;
  static constexpr uint32_t QB = NH * NC * 128;  // one Q buffer
  static constexpr uint32_t PB = 2 * NC * 128;   // one P^T buffer's high or low parts
  static constexpr uint32_t Q = NS * TILE;       // two buffers: the next piece's Q comes early
  static constexpr uint32_t P = Q + 2 * QB;
  static constexpr uint32_t RED = P + 4 * PB;    // float [4][NC]
  static constexpr uint32_t SUMS = RED + 4 * NC * 4;  // float [NC][kSumStride]
  static constexpr uint32_t BARS = SUMS + NC * kSumStride * 4;
  // (at HD = 64 an MMA's second 64-wide block lies one half tile further on, past the last stage's end)
  static constexpr uint32_t TOTAL = BARS + 512 + 1024 + (HD == 64 ? kHalf : 0);
};

struct FewBars {
  uint64_t full[10], empty[10], q_full[2], q_empty[2], s_full[2], s_empty[2], p_full[2], p_empty[2], o_full, o_empty, drain;
  uint32_t tmem;
  int abort, never;
};
static_assert(sizeof(FewBars) <= 512, "FewBars outgrew its place");

static_assert(FewLayout<128, 16>::TOTAL <= 232448 && FewLayout<128, 32>::TOTAL <= 232448 &&
                  FewLayout<64, 16>::TOTAL <= 232448 && FewLayout<64, 32>::TOTAL <= 232448,
              "more shared memory than a block can have");
// The library's kernels with TMEM take 48 KB of shared memory or more, an SM has 228 KB.
static_assert(FewLayout<128, 16>::TOTAL > 180 * 1024 && FewLayout<128, 32>::TOTAL > 180 * 1024 &&
                  FewLayout<64, 16>::TOTAL > 180 * 1024 && FewLayout<64, 32>::TOTAL > 180 * 1024,
              "a kernel that waits for TMEM could share an SM with blocks that hold some and wait for it");

// Kept scores: [KV head][key][score_floats(rows of the group)] for every group of
// tokens, rows rounded up to whole vectors.  A token has room for the rounded
// rows of its own, which suffices for groups of any size.
__host__ __device__ __forceinline__ int score_floats(int rows) { return (rows + 3) & ~3; }
__device__ __forceinline__ int64_t score_index(const AttnParams& p, const ChunkPlan& c, int64_t tok, int kvh, int key, int rows) {
  return tok * p.hkv * p.len_k * score_floats(c.group) + ((int64_t)kvh * p.len_k + key) * score_floats(rows);
}

__device__ __forceinline__ void fail(const AttnParams& p, FewBars* s) {
  s->abort = 1;
  if (p.dev_status) atomicCAS(p.dev_status, kDevOk, kDevWaitTimeout);
}

template <int HD, bool BF16, int NC>
__global__ void __launch_bounds__(kFewThreads, 1)
    few_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttnParams p, const __grid_constant__ ChunkPlan c,
               const __grid_constant__ PieceWs ws, float* scores) {
  using L = FewLayout<HD, NC>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  constexpr int NH = L::NH, NS = L::NS;
  constexpr uint32_t IDESC_QK = idesc_f16(BF16, 128, NC, false, false);
  constexpr uint32_t IDESC_PV = idesc_f16(BF16, 128, NC, true, false);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  FewBars* bars = reinterpret_cast<FewBars*>(smem + L::BARS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  allow_dependents();
  if (warp == 4 && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars->q_full[s], 1);
      mbar_init(&bars->q_empty[s], 1);
      mbar_init(&bars->s_full[s], 1);
      mbar_init(&bars->s_empty[s], 4);
      mbar_init(&bars->p_full[s], 4);
      mbar_init(&bars->p_empty[s], 1);
    }
    mbar_init(&bars->o_full, 1);
    mbar_init(&bars->o_empty, 4);
    mbar_init(&bars->drain, 1);
    bars->abort = bars->never = 0;
    fence_barrier_init();
  }
  // (TMEM held while waiting for the predecessor: one that still has to allocate
  // its own cannot be on this SM, see the assertion on FewLayout)
  if (warp == 5) tmem_alloc(&bars->tmem, 128);
  wait_for_predecessor();
  Walk walk(p, c.tpb);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;  // S^T buffers at 0 and NC, O^T at 2 NC
  volatile int* abort_flag = &bars->abort;

  if (warp == 4) {
    // ------------------------------------------------------------ producer
    bool ok = true;
    int issued = 0, pieces = 0;
    while (ok && walk.next()) {
      const Unit& u = walk.u;
      const int qb = pieces & 1;
      int row = tile_box_row(p, c, u.b, u.g.k_len, walk.piece.kt0);
      if (!(ok = wait_warp(&bars->q_empty[qb], ((pieces >> 1) & 1) ^ 1, abort_flag))) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars->q_full[qb], NH * c.tpb * c.group * 128);
        for (int hh = 0; hh < NH; ++hh)
          tma_load_4d(smem + L::Q + qb * L::QB + hh * NC * 128, &tm_q, &bars->q_full[qb], 64 * hh, u.kvh * c.group,
                      u.g.q_start + u.tok0, 0);
      }
      ++pieces;
      for (int t = 0; t < walk.piece.nt && ok; ++t) {
        const int next = t + 1 < walk.piece.nt ? tile_box_row(p, c, u.b, u.g.k_len, walk.piece.kt0 + t + 1) : -1;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int st = issued % NS;
          if (!(ok = wait_warp(&bars->empty[st], ((issued / NS) & 1) ^ 1, abort_flag))) break;
          load_key_tile_tma<NH>(smem + st * L::TILE, kv ? &tm_v : &tm_k, &bars->full[st], row, c.box_rows, u.kvh);
          ++issued;
        }
        row = next;
      }
    }
    if (!ok && lane == 0) {
      fail(p, bars);
      for (int i = max(0, pieces - 2); i < pieces; ++i) mbar_wait(&bars->q_full[i & 1], (i >> 1) & 1, &bars->never);
      for (int i = max(0, issued - NS); i < issued; ++i) mbar_wait(&bars->full[i % NS], (i / NS) & 1, &bars->never);
    }
    __syncwarp();
  } else if (warp == 5) {
    // ------------------------------------------------------------ MMA issuer
    // Items of the ring: K of tile it is 2 it, V is 2 it + 1 (it runs over all pieces).
    bool ok = true;
    int it = 0, pieces = 0;
    const uint32_t base = smem_u32(smem);
    auto issue_s = [&](int i, int qb, bool last) -> bool {
      const int item = 2 * i, st = item % NS, sb = i & 1;
      if (!wait_warp(&bars->full[st], (item / NS) & 1, abort_flag)) return false;
      if (!wait_warp(&bars->s_empty[sb], ((i >> 1) & 1) ^ 1, abort_flag)) return false;
      tc_fence_after();
      const uint64_t k_desc = sw128_desc(base + st * L::TILE, 16, 1024), q_desc = sw128_desc(base + L::Q + qb * L::QB, 16, 1024);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_f16_ss(tmem + sb * NC, desc_at(k_desc, (kk >> 2) * kHalf + (kk & 3) * 32),
                     desc_at(q_desc, (kk >> 2) * NC * 128 + (kk & 3) * 32), IDESC_QK, kk > 0);
        mma_commit(&bars->s_full[sb]);
        mma_commit(&bars->empty[st]);
        if (last) mma_commit(&bars->q_empty[qb]);
      }
      __syncwarp();
      return true;
    };
    while (walk.next()) {
      const int nt = walk.piece.nt, qb = pieces & 1;
      if (ok) ok = wait_warp(&bars->q_full[qb], (pieces >> 1) & 1, abort_flag) && issue_s(it, qb, nt == 1);
      for (int t = 0; t < nt && ok; ++t, ++it) {
        if (t + 1 < nt && !(ok = issue_s(it + 1, qb, t + 2 == nt))) break;
        const int item = 2 * it + 1, st = item % NS, pb = it & 1;
        if (t == 0 && !(ok = wait_warp(&bars->o_empty, (pieces & 1) ^ 1, abort_flag))) break;
        if (!(ok = wait_warp(&bars->full[st], (item / NS) & 1, abort_flag))) break;
        if (!(ok = wait_warp(&bars->p_full[pb], (it >> 1) & 1, abort_flag))) break;
        tc_fence_after();
        const uint64_t v_desc = sw128_desc(base + st * L::TILE, kHalf, 1024), p_desc = sw128_desc(base + L::P + pb * 2 * L::PB, 16, 1024);
        if (elect_one()) {
          // A = V^T: rows of the tile are keys (the K axis), head dims contiguous;
          // at HD = 64 rows 64 .. 127 of the product come from the bytes after
          // the tile and are not read
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int kk = 0; kk < kTileKeys / 16; ++kk)
              mma_f16_ss(tmem + 2 * NC, desc_at(v_desc, kk * 16 * 128),
                         desc_at(p_desc, part * L::PB + (kk >> 2) * NC * 128 + (kk & 3) * 32), IDESC_PV,
                         t > 0 || part > 0 || kk > 0);
          mma_commit(&bars->empty[st]);
          mma_commit(&bars->p_empty[pb]);
          if (t + 1 == nt) mma_commit(&bars->o_full);
        }
        __syncwarp();
      }
      ++pieces;
    }
    if (lane == 0 && !ok) {
      fail(p, bars);
      mma_commit(&bars->drain);
      mbar_wait(&bars->drain, 0, &bars->never);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax
    const int r = threadIdx.x;  // key of the tile; head dim of O^T
    if (blockIdx.x == gridDim.x - 1) record_bad_offsets(p, r, 128);
    const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
    const float zs = p.scale * kLog2e;
    float* red = reinterpret_cast<float*>(smem + L::RED);
    float* sums = reinterpret_cast<float*>(smem + L::SUMS);
    const uint32_t p_base = smem_u32(smem + L::P);
    // this key's 16-byte chunk of a P^T row, before the row's swizzle
    const uint32_t p_half = (uint32_t)(r >> 6) * NC * 128, p_chunk = (uint32_t)((r >> 3) & 7), p_in = (uint32_t)(r & 7) * 2;
    bool ok = true;
    int it = 0, pieces = 0;
    while (walk.next()) {
      const Unit& u = walk.u;
      const Piece& pc = walk.piece;
      const int rows = u.ntok * c.group;
      const int keep = score_floats(rows);
      float* kept = scores + score_index(p, c, u.g.q_start + u.tok0, u.kvh, 0, rows);
      float m[NC], l[NC];
#pragma unroll
      for (int x = 0; x < NC; ++x) m[x] = l[x] = 0.f;
      for (int t = 0; t < pc.nt; ++t, ++it) {
        const int sb = it & 1, kb = (pc.kt0 + t) * kTileKeys, key = kb + r;
        if (ok) ok = wait_warp(&bars->s_full[sb], (it >> 1) & 1, abort_flag);
        tc_fence_after();
        uint32_t sx[NC];
        if constexpr (NC == 16) tmem_ld16(tmem + lane_addr + sb * NC, sx);
        else tmem_ld32(tmem + lane_addr + sb * NC, sx);
        tmem_wait_ld();
        tc_fence_before();
        warp_arrive(&bars->s_empty[sb]);
        // rows that see this key: all of them before the first token's limit
        int lo = 0;
        if (p.causal) lo = max(0, key - u.g.shift - u.tok0) * c.group;
        if (key >= u.g.k_len) lo = NC;
        float x[NC];
        bool high = false;
#pragma unroll
        for (int e = 0; e < NC; ++e) {
          x[e] = e >= lo && e < rows ? __uint_as_float(sx[e]) * zs : kNegInf;
          high |= x[e] > m[e] + kRescale<BF16>;
        }
        if (scores != nullptr && key < u.g.k_len) {
          float4* dst = reinterpret_cast<float4*>(kept + (int64_t)key * keep);
#pragma unroll
          for (int e = 0; e < NC; e += 4)
            if (e < keep) dst[e / 4] = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        }
        if (!BF16 && t == 0) {
          // rows that the warp's keys leave below the implicit zero logit
          uint32_t seen = 0u, above = 0u;
#pragma unroll
          for (int e = 0; e < NC; ++e) {
            seen |= x[e] > kNegInf ? 1u << e : 0u;
            above |= x[e] >= 0.f ? 1u << e : 0u;
          }
          high |= (__reduce_or_sync(0xffffffffu, seen) & ~__reduce_or_sync(0xffffffffu, above)) != 0u;
        }
        if (named_bar_or(1, 128, high)) {
          // some row passed its reference (float16: or may start far below it): the tile's row maxima over the four warps
#pragma unroll
          for (int e = 0; e < NC; ++e) {
            // bfloat16: only maxima above m + 2^3 > 0 matter, and positive floats compare as integers
            const int w = __reduce_max_sync(0xffffffffu, BF16 ? __float_as_int(fmaxf(x[e], 0.f)) : ordered_int(x[e]));
            if (lane == 0) red[warp * NC + e] = __int_as_float(BF16 ? w : ordered_int(__int_as_float(w)));
          }
          named_bar_sync(1, 128);
          float alpha[NC];
#pragma unroll
          for (int e = 0; e < NC; ++e) {
            const float top = fmaxf(fmaxf(red[e], red[NC + e]), fmaxf(red[2 * NC + e], red[3 * NC + e]));
            alpha[e] = 1.f;
            if (top > m[e] + kRescale<BF16> || (!BF16 && t == 0)) {
              const float ref = BF16 ? top : reference16(top);
              alpha[e] = exp2f(m[e] - ref);
              m[e] = ref;
              l[e] *= alpha[e];
            }
          }
          named_bar_sync(1, 128);  // red may be written again
          if (t > 0) {
            // O^T holds every earlier tile once P V of the last one is done
            if (ok) ok = wait_warp(&bars->p_empty[sb ^ 1], ((it - 1) >> 1) & 1, abort_flag);
            tc_fence_after();
            uint32_t o[NC];
            if constexpr (NC == 16) tmem_ld16(tmem + lane_addr + 2 * NC, o);
            else tmem_ld32(tmem + lane_addr + 2 * NC, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < NC; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha[e]);
            if constexpr (NC == 16) tmem_st16(tmem + lane_addr + 2 * NC, o);
            else tmem_st32(tmem + lane_addr + 2 * NC, o);
            tmem_wait_st();
          }
        }
        if (ok) ok = wait_warp(&bars->p_empty[sb], ((it >> 1) & 1) ^ 1, abort_flag);
        const uint32_t dst = p_base + sb * 2 * L::PB + p_half + p_in;
#pragma unroll
        for (int e = 0; e < NC; ++e) {
          const float v = ex2_ftz(x[e] - m[e]);
          l[e] += v;
          const T hi = from_f32<T>(v), lo = from_f32<T>(v - to_f32<T>(hi));
          const uint32_t at = dst + e * 128 + ((p_chunk ^ (e & 7)) << 4);
          sts_u16(at, *reinterpret_cast<const uint16_t*>(&hi));
          sts_u16(at + L::PB, *reinterpret_cast<const uint16_t*>(&lo));
        }
        if (kb + kTileKeys > u.g.k_len) {
          // V rows past the sequence: zeroed, since 0 x NaN would reach O
          const int item = 2 * it + 1, st = item % NS, tail = max(u.g.k_len - kb, 0);
          if (ok) ok = wait_warp(&bars->full[st], (item / NS) & 1, abort_flag);
          for (int y = r; ok && y < (kTileKeys - tail) * 8 * NH; y += 128) {
            const int hh = y / ((kTileKeys - tail) * 8), z = y - hh * (kTileKeys - tail) * 8;
            *reinterpret_cast<uint4*>(smem + st * L::TILE + hh * kHalf + tail * 128 + z * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        warp_arrive(&bars->p_full[sb]);
      }
      // ---- the piece's result
      if (ok) ok = wait_warp(&bars->o_full, pieces & 1, abort_flag);
      tc_fence_after();
      uint32_t o[NC];
      if constexpr (NC == 16) tmem_ld16(tmem + lane_addr + 2 * NC, o);
      else tmem_ld32(tmem + lane_addr + 2 * NC, o);
      tmem_wait_ld();
      tc_fence_before();
      warp_arrive(&bars->o_empty);
      // sums of l over the keys' threads: eight lanes add up a row's 128 values
#pragma unroll
      for (int e = 0; e < NC; ++e) sums[e * kSumStride + r] = l[e];
      named_bar_sync(1, 128);
#pragma unroll
      for (int e0 = 0; e0 < NC; e0 += 16) {
        const float4* s4 = reinterpret_cast<const float4*>(sums + (e0 + (r >> 3)) * kSumStride + (r & 7) * 16);
        float w = 0.f;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float4 v = s4[y];
          w += (v.x + v.y) + (v.z + v.w);
        }
#pragma unroll
        for (int y = 4; y > 0; y >>= 1) w += __shfl_xor_sync(0xffffffffu, w, y);
        if ((r & 7) == 0) red[e0 + (r >> 3)] = w;
      }
      named_bar_sync(1, 128);
      int64_t tok = u.g.q_start + u.tok0;
      int h = u.kvh * c.group;
#pragma unroll
      for (int e = 0; e < NC; ++e) {
        if (e < rows) {
          const float sum = red[e];
          if (pc.whole) {
            const RowEnd end = end_of_row<BF16>(m[e], sum);
            if (r < HD)
              static_cast<T*>(p.o)[tok * p.o_st + (int64_t)h * p.o_sh + r] = from_f32<T>(__uint_as_float(o[e]) * end.inv);
            if (r == 0) {
              p.stats[(int64_t)h * p.rows_total + tok] = end.m;
              p.stats[(int64_t)(p.hq + h) * p.rows_total + tok] = end.l;
            }
          } else {
            const int64_t at = (int64_t)pc.slot * ws.rows + e;
            if (r < HD) ws.o[at * HD + r] = __uint_as_float(o[e]);
            if (r == 0) ws.ml[at] = make_float2(m[e], sum);
          }
          if (++h == (u.kvh + 1) * c.group) {
            h = u.kvh * c.group;
            ++tok;
          }
        }
      }
      if (pc.kt0 == 0 && r < u.ntok)
        ws.info[(int64_t)(u.g.q_start + u.tok0 + r) * p.hkv + u.kvh] = make_int4(pc.u0, u.tiles, r * c.group, walk.quota);
      named_bar_sync(1, 128);  // red may be written again
      ++pieces;
    }
    if (!ok && lane == 0) fail(p, bars);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, 128);
  }
}

// Key weights from the kept scores: thread = key of a (token group, KV head).
template <int NC>
__global__ void __launch_bounds__(256) few_weights_kernel(const AttnParams p, const ChunkPlan c, const float* scores,
                                                          float* kw, int64_t ldw) {
  allow_dependents();
  wait_for_predecessor();
  __shared__ float consts[NC];
  const int b = blockIdx.z, kvh = blockIdx.y, key = blockIdx.x * 256 + threadIdx.x;
  const Geometry g = geometry(p, b);
  if (blockIdx.x * 256 >= g.k_len) return;
  float sum = 0.f;
  for (int tok0 = 0; tok0 < g.q_len; tok0 += c.tpb) {
    const int rows = min(c.tpb, g.q_len - tok0) * c.group;
    __syncthreads();
    if (threadIdx.x < NC) {
      const int e = threadIdx.x;
      float k = kNegInf;
      if (e < rows) {
        const int64_t si = stat_index(p, g, kvh * c.group + e % c.group, tok0 + e / c.group);
        k = -(p.stats[si] + log2f(p.stats[(int64_t)p.hq * p.rows_total + si]));
      }
      consts[e] = k;
    }
    __syncthreads();
    // keys that no row of the group sees have no tile, hence no scores
    if (key >= g.k_len || (p.causal && key > g.shift + tok0 + rows / c.group - 1)) continue;
    const float4* s = reinterpret_cast<const float4*>(scores + score_index(p, c, g.q_start + tok0, kvh, key, rows));
#pragma unroll
    for (int e = 0; e < NC; e += 4) {
      if (e >= rows) break;
      const float4 x = s[e / 4];
      sum += ex2_ftz(x.x + consts[e]) + ex2_ftz(x.y + consts[e + 1]) + ex2_ftz(x.z + consts[e + 2]) +
             ex2_ftz(x.w + consts[e + 3]);
    }
  }
  if (key < g.k_len) {
    const int64_t tok = key_token(p, g, b, key);
    if (tok >= 0) atomicAdd(kw + (int64_t)kvh * ldw + tok, sum);
  }
}

// ------------------------------------------------------------------ host
template <int HD, bool BF16, int NC>
cudaError_t run(const AttnParams& p, const ChunkPlan& c, float* kw, int64_t ldw, void* workspace, cudaStream_t s) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  CUtensorMap tq, tk, tv;
  if (!make_row_map(&tq, p, BF16, c) || !make_page_map(&tk, p.k, p.k_st, p.k_sh, p, BF16, c) ||
      !make_page_map(&tv, p.v, p.v_st, p.v_sh, p, BF16, c))
    return cudaErrorInvalidValue;
  const int ctas = sm_count();
  const PieceWs ws = piece_ws(p, ctas, NC, workspace);
  float* scores = kw == nullptr ? nullptr
                                : reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + piece_layout(p, ctas, NC).total);
  constexpr int smem = FewLayout<HD, NC>::TOTAL;
  cudaError_t e = allow_smem<few_kernel<HD, BF16, NC>>(smem);
  if (e != cudaSuccess) return e;
  e = launch_dependent(few_kernel<HD, BF16, NC>, dim3(ctas), kFewThreads, smem, s, tq, tk, tv, p, c, ws, scores);
  if (e != cudaSuccess) return e;
  e = launch_dependent(combine_pieces_kernel<HD, T>, dim3(p.rows_total * p.hkv), 128, 0, s, p, ws, c.group);
  if (e != cudaSuccess || kw == nullptr || p.len_k == 0) return e;
  return launch_dependent(few_weights_kernel<NC>, dim3((p.len_k + 255) / 256, p.hkv, p.batch), 256, 0, s, p, c,
                          static_cast<const float*>(scores), kw, ldw);
}

// MMA columns for at most 32 packed rows.
int few_columns(const AttnParams& p) {
  const int64_t n = p.len_q < p.rows_total ? p.len_q : p.rows_total;
  const int64_t rows = n * (p.hq / p.hkv);
  return rows <= 16 ? 16 : (rows <= 32 ? 32 : 0);
}

}  // namespace

// Scores kept at most; beyond, the weights read K again.  A bound on memory, not
// on time: kept scores stay ahead (0.25 GiB, 64 x 1 token on 32k keys: 1504
// against 3278 us; 0.5 GiB, 64 x 8 tokens on 8k: 726 against 818).
constexpr int64_t kFewScoreBytes = 1ll << 30;

static int64_t score_bytes(const AttnParams& p, const ChunkPlan& c) {
  return (int64_t)p.rows_total * p.hkv * p.len_k * score_floats(c.group) * 4;
}

// Against the dense kernel, both measured (8 KV heads, us, few / dense): up to 16
// packed rows ahead everywhere (1 token on 32k keys 49 / 51, 32 x 1 on 8k 194 /
// 213, 16 x 4 tokens of 4 heads on 8k 115 / 121; with weights 54 / 82, 220 / 442,
// 148 / 238).  17 to 32 rows: behind without weights (16 x 4 tokens of 8 heads on
// 8k 125 / 117, 1 x 4 on 32k 70 / 59), mostly ahead with them (217 / 235, 104 /
// 89); they run here for P in two parts.
bool chunk_few_applies(const AttnParams& p, const ChunkPlan& c, bool weights) {
  if (p.norm != HFAN_SOFTMAX1 || few_columns(p) == 0) return false;
  return !weights || score_bytes(p, c) <= kFewScoreBytes;
}

int64_t chunk_few_workspace(const AttnParams& p, const ChunkPlan& c, bool weights) {
  return piece_layout(p, sm_count(), few_columns(p)).total + (weights ? score_bytes(p, c) : 0);
}

cudaError_t chunk_few_fwd(int dtype, const AttnParams& p, const ChunkPlan& c, float* kw, int64_t ldw, void* workspace,
                          cudaStream_t s) {
  const bool bf16 = dtype == HFAN_BFLOAT16;
  if (few_columns(p) == 16) {
    if (p.d == 128) return bf16 ? run<128, true, 16>(p, c, kw, ldw, workspace, s) : run<128, false, 16>(p, c, kw, ldw, workspace, s);
    return bf16 ? run<64, true, 16>(p, c, kw, ldw, workspace, s) : run<64, false, 16>(p, c, kw, ldw, workspace, s);
  }
  if (p.d == 128) return bf16 ? run<128, true, 32>(p, c, kw, ldw, workspace, s) : run<128, false, 32>(p, c, kw, ldw, workspace, s);
  return bf16 ? run<64, true, 32>(p, c, kw, ldw, workspace, s) : run<64, false, 32>(p, c, kw, ldw, workspace, s);
}

}  // namespace hfan
