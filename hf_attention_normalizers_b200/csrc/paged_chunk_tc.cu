// Attention of a ragged chunk of new tokens over a paged cache, on tcgen05
// tensor cores (16-bit inputs, head_dim 64 / 128, pages of a multiple of 8
// tokens, positive scale).
//
// A unit of work is two tiles of 128 packed (token, head) rows of one sequence
// and KV head; a CTA takes pieces of units (paged_walk.cuh) in tiles of 128
// keys that TMA fetches straight from the pages (one box per page or per 128
// rows of it):
//
//   warps 0-3, 4-7  row warps of tile 0 / 1: thread = TMEM lane = row.  A
//                   thread reads its whole S row, so the running maximum and
//                   sum need no exchange, and writes P over S as packed
//                   16-bit pairs (the A operand of P V).
//   warp 8          producer: Q of a piece, then K0 V0 K1 V1 ... through one ring.
//   warps 9, 10     MMA issuers of tile 0 / 1.
//
// The two tiles are independent chains that share the K and V stages.  A chain
// works in halves of a key tile (64 keys) with two S buffers: while the row
// warps exponentiate half j, the tensor pipe has S of j + 1 ready and works on
// O += P V of j - 1 and S of j + 1 into the buffer that P of j - 1 leaves, so
// neither side waits for the other's latency.  (One 128-key S buffer a chain,
// all that fits beside O, left the row warps waiting 1700 of 4600 cycles.)
// softmax1 exponentiates against a reference m that need not be the maximum:
// while the exponentials of a half sum up to at most 2^12, O loses nothing by
// it, and no maximum is taken at all.  A row that passes it moves m to its
// maximum.  m starts at the implicit zero logit in bfloat16, whose exponents
// reach as far as float32's, so that P loses nothing on the low side either; in
// float16 it starts 2^8 below the maximum of the piece's first half and moves
// past a sum of 2^15, see reference16 (paged_walk.cuh).
//
// P is rounded to the inputs' type, at most half a unit of each p beside the
// rounding of the result: a second 16-bit part for the rest would repeat the
// P V products, half of the tensor pipe's work here.
//
// Measured: 1024 tokens on 32k keys (32 / 8 heads of 128), 0.55 TFLOP: 0.52 ms
// from a cool start, 0.64 ms in a row, where the 1000 W limit holds the clock at
// 1.6 GHz; tensor pipe busy 49% of the cycles.  Passing tiles through without
// any row arithmetic takes 0.43 ms: N = 64 products read Q twice as often, which
// makes them wait for shared memory (48 cycles instead of 32), the price of the
// second S buffer.  Loads alone take 0.22 ms.
//
// sparsemax / entmax15 come here with their thresholds known, for the units
// that the scan (paged_chunk_sparse.cu) could not serve from its buffers.
#include <cuda.h>

#include "common.cuh"
#include "paged_chunk.cuh"
#include "paged_serving.cuh"
#include "paged_walk.cuh"
#include "params.cuh"
#include "tc_common.cuh"
#include "tc_ptx.cuh"

namespace hfan {
namespace {

using namespace tc;

constexpr int kChunkThreads = 352;
constexpr int kMaxRing = 8;
// (bfloat16, a mixed batch of 452 tokens / 4 x 256 on 8k keys, us: 2^4 100 / 183,
// 2^8 90 / 162, 2^12 91 / 161, 2^20 91 / 161; scores of four times unit
// deviation: 106 / 200, 100 / 187, 95 / 170, 99 / 194)
template <bool BF16>
constexpr float kHighSum = BF16 ? 4096.f : 32768.f;  // (also keeps P below float16's 65504)
// Factor of s - tau: float16 takes the sparse normalizers' P (at most 1) times
// 2^14, since supports of tens of thousands of keys lie among its subnormals.
template <bool BF16, int NORM>
constexpr float kLift = BF16 ? 1.f : (NORM == HFAN_SPARSEMAX ? 0x1p14f : 0x1p7f);
constexpr int kUnitRows = 2 * kTileRows;
constexpr int kHalfKeys = kTileKeys / 2;

template <int HD>
constexpr int chunk_ring() { return HD == 128 ? 5 : 8; }

struct ChunkBars {
  uint64_t q_full, q_empty, full[kMaxRing], empty[kMaxRing];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2], o_empty[2], drain[2];
};
struct ChunkCtl {
  uint32_t tmem;
  int abort, never;  // never stays 0: the abort flag of waits that must not be cut short
};

template <int HD>
struct ChunkLayout {
  static constexpr int NH = HD / 64, NS = chunk_ring<HD>();
  static constexpr uint32_t TILE = NH * kHalf;
  static constexpr uint32_t RING = 2 * TILE;
  static constexpr uint32_t BARS = RING + NS * TILE;
  static constexpr uint32_t CTL = BARS + sizeof(ChunkBars);
  static constexpr uint32_t TOTAL = CTL + sizeof(ChunkCtl) + 1024;
};

__device__ __forceinline__ void fail(const AttnParams& p, ChunkCtl* ctl) {
  ctl->abort = 1;
  if (p.dev_status) atomicCAS(p.dev_status, kDevOk, kDevWaitTimeout);
}

// The sparse normalizers' source of work: the unit of the block's grid
// coordinates, when the scan has left its output to this kernel.
class FlaggedUnit {
 public:
  Unit u;
  Piece piece;
  static constexpr int quota = 1;
  __device__ __forceinline__ FlaggedUnit(const AttnParams& p, int per, const int* flags) {
    int group;
    left_ = find_group(p, per, blockIdx.x, &u.b, &group) && flags[blockIdx.x * p.hkv + blockIdx.y] != 0;
    if (!left_) return;
    u.g = geometry(p, u.b);
    u.kvh = blockIdx.y;
    u.tok0 = group * per;
    u.ntok = min(per, u.g.q_len - u.tok0);
    const int k_hi = p.causal ? min(u.g.k_len, u.tok0 + u.ntok + u.g.shift) : u.g.k_len;
    u.tiles = max((k_hi + kTileKeys - 1) / kTileKeys, 1);
    piece = Piece{0, u.tiles, 0, 0, true};
  }
  __device__ __forceinline__ bool any() const { return left_; }
  __device__ __forceinline__ bool next() {
    const bool r = left_;
    left_ = false;
    return r;
  }

 private:
  bool left_;
};

class Stretch : public Walk {
 public:
  __device__ __forceinline__ Stretch(const AttnParams& p, int per, const int*) : Walk(p, per) {}
  __device__ __forceinline__ bool any() const { return true; }
};

template <int HD, bool BF16, int NORM>
__global__ void __launch_bounds__(kChunkThreads, 1)
    chunk_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttnParams p,
                     const __grid_constant__ ChunkPlan c, const __grid_constant__ PieceWs ws, const int* flags) {
  using L = ChunkLayout<HD>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  using Source = typename std::conditional<NORM == HFAN_SOFTMAX1, Stretch, FlaggedUnit>::type;
  constexpr int NH = L::NH, NS = L::NS;
  constexpr uint32_t IDESC_QK = idesc_f16(BF16, 128, kHalfKeys, false, false);
  constexpr uint32_t IDESC_PV = idesc_f16(BF16, 128, HD, false, true);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  ChunkBars* bars = reinterpret_cast<ChunkBars*>(smem + L::BARS);
  ChunkCtl* ctl = reinterpret_cast<ChunkCtl*>(smem + L::CTL);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  allow_dependents();
  if (warp == 8 && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_empty, 2);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 2);
    }
    for (int s = 0; s < 2; ++s) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bars->s_full[s][h], 1);
        mbar_init(&bars->p_full[s][h], 4);
      }
      mbar_init(&bars->pv_done[s], 1);
      mbar_init(&bars->o_empty[s], 4);
      mbar_init(&bars->drain[s], 1);
    }
    ctl->abort = ctl->never = 0;
    fence_barrier_init();
  }
  wait_for_predecessor();
  Source src(p, 2 * c.tpb, flags);
  if (!src.any()) return;  // nothing was left to this block
  if (warp == 8) tmem_alloc(&ctl->tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;  // S of tile 0 (two halves) | of tile 1 | O0 | O1, 128 columns each
  volatile int* abort_flag = &ctl->abort;

  if (warp >= 8) {
    if (warp == 8) {
      // ---------------------------------------------------------- producer
      bool ok = true;
      int st = 0, ph = 1, issued = 0, pieces = 0;
      while (ok && src.next()) {
        const Unit& u = src.u;
        const int nact = u.ntok > c.tpb ? 2 : 1;  // tiles with rows
        int row = tile_box_row(p, c, u.b, u.g.k_len, src.piece.kt0);
        if (!(ok = wait_warp(&bars->q_empty, (pieces & 1) ^ 1, abort_flag))) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars->q_full, nact * NH * c.tpb * c.group * 128);
          for (int q = 0; q < nact; ++q)
            for (int hh = 0; hh < NH; ++hh)
              tma_load_4d(smem + q * L::TILE + hh * kHalf, &tm_q, &bars->q_full, 64 * hh, u.kvh * c.group,
                          u.g.q_start + u.tok0 + q * c.tpb, 0);
        }
        ++pieces;
        for (int t = 0; t < src.piece.nt && ok; ++t) {
          const int next = t + 1 < src.piece.nt ? tile_box_row(p, c, u.b, u.g.k_len, src.piece.kt0 + t + 1) : -1;
#pragma unroll
          for (int kv = 0; kv < 2 && ok; ++kv) {
            if (!(ok = wait_warp(&bars->empty[st], ph, abort_flag))) break;
            load_key_tile_tma<NH>(smem + L::RING + st * L::TILE, kv ? &tm_v : &tm_k, &bars->full[st], row, c.box_rows, u.kvh);
            ++issued;
            if (++st == NS) {
              st = 0;
              ph ^= 1;
            }
          }
          row = next;
        }
      }
      if (!ok && lane == 0) {
        fail(p, ctl);
        // its own copies land before the CTA leaves
        if (pieces > 0) mbar_wait(&bars->q_full, (pieces - 1) & 1, &ctl->never);
        for (int i = max(0, issued - NS); i < issued; ++i) mbar_wait(&bars->full[i % NS], (i / NS) & 1, &ctl->never);
      }
      __syncwarp();
    } else {
      // ---------------------------------------------------------- MMA issuers
      // (the whole warp walks the loops and one elected lane issues: a branch
      // for lane 0 around them made every MMA dearer to issue, 538 against 508 us)
      const int q = warp - 9;
      const uint32_t q_base = smem_u32(smem + q * L::TILE), ring = smem_u32(smem + L::RING);
      const uint32_t s_col = tmem + q * 128, o_col = tmem + 256 + q * 128;
      const uint64_t q_desc = sw128_desc(q_base, 16, 1024);
      bool ok = true;
      int items = 0, pieces = 0, mine = 0;  // ring items and pieces so far; pieces in which this tile has rows
      int jj = 0;                           // halves of those pieces
      while (src.next()) {
        const int nt = src.piece.nt;
        if (ok) {
          ok = wait_warp(&bars->q_full, pieces & 1, abort_flag);
          if (q == 1 && src.u.ntok <= c.tpb) {
            // no rows: the stages are only passed on
            for (int x = items; x < items + 2 * nt && ok; ++x) {
              if (!(ok = wait_warp(&bars->full[x % NS], (x / NS) & 1, abort_flag))) break;
              if (lane == 0) mbar_arrive(&bars->empty[x % NS]);
            }
            if (lane == 0) mbar_arrive(&bars->q_empty);
          } else {
            // S of half j into buffer j & 1, which P V of half j - 2 has left
            auto issue_s = [&](int j) -> bool {
              const int item = items + 2 * (j >> 1), st = item % NS, h = j & 1;
              if (h == 0 && !wait_warp(&bars->full[st], (item / NS) & 1, abort_flag)) return false;
              tc_fence_after();
              const uint64_t k_desc = sw128_desc(ring + st * L::TILE + h * kHalfKeys * 128, 16, 1024);
              if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                  const uint32_t o = (kk >> 2) * kHalf + (kk & 3) * 32;
                  mma_f16_ss(s_col + h * kHalfKeys, desc_at(q_desc, o), desc_at(k_desc, o), IDESC_QK, kk > 0);
                }
                mma_commit(&bars->s_full[q][h]);
                if (h == 1) mma_commit(&bars->empty[st]);
                if (j == 2 * nt - 1) mma_commit(&bars->q_empty);
              }
              __syncwarp();
              return true;
            };
            ok = ok && issue_s(0) && issue_s(1);
            for (int j = 0; j < 2 * nt && ok; ++j, ++jj) {
              const int item = items + 2 * (j >> 1) + 1, st = item % NS, h = j & 1;
              if (h == 0 && !(ok = wait_warp(&bars->full[st], (item / NS) & 1, abort_flag))) break;
              if (j == 0 && !(ok = wait_warp(&bars->o_empty[q], (mine & 1) ^ 1, abort_flag))) break;
              if (!(ok = wait_warp(&bars->p_full[q][h], (jj >> 1) & 1, abort_flag))) break;
              tc_fence_after();
              const uint64_t v_desc = sw128_desc(ring + st * L::TILE + h * kHalfKeys * 128, kHalf, 1024);
              if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < kHalfKeys / 16; ++kk)
                  mma_f16_ts(o_col, s_col + h * kHalfKeys + kk * 8, desc_at(v_desc, kk * 16 * 128), IDESC_PV, j > 0 || kk > 0);
                mma_commit(&bars->pv_done[q]);
                if (h == 1) mma_commit(&bars->empty[st]);
              }
              __syncwarp();
              if (j + 2 < 2 * nt) ok = issue_s(j + 2);
            }
            ++mine;
          }
        }
        items += 2 * nt;
        ++pieces;
        __syncwarp();
      }
      if (lane == 0 && !ok) {
        fail(p, ctl);
        mma_commit(&bars->drain[q]);
        mbar_wait(&bars->drain[q], 0, &ctl->never);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ row warps
    const int q = warp >> 2, r = threadIdx.x & 127;
    if (NORM == HFAN_SOFTMAX1 && blockIdx.x == gridDim.x - 1) record_bad_offsets(p, threadIdx.x, 256);
    const int rt = r / c.group, rg = r - rt * c.group;  // token of the tile, head of the group
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lane_addr + q * 128, o_col = tmem + lane_addr + 256 + q * 128;
    const float zs = NORM == HFAN_SOFTMAX1 ? p.scale * kLog2e : (NORM == HFAN_SPARSEMAX ? p.scale : 0.5f * p.scale);
    bool ok = true;
    int jj = 0;     // halves so far
    int items = 0;  // ring items of the pieces before this one
    while (src.next()) {
      const Unit& u = src.u;
      const Piece& pc = src.piece;
      const int v0 = items + 1;  // item of the piece's first V tile
      items += 2 * pc.nt;
      if (q == 1 && u.ntok <= c.tpb) continue;
      const int tl = q * c.tpb + rt, i = u.tok0 + tl;  // token of the unit, of the sequence
      const bool row_ok = rt < c.tpb && tl < u.ntok;
      const int h = u.kvh * c.group + rg;
      // visible keys [0, vis)
      int vis = row_ok ? u.g.k_len : 0;
      if (p.causal && row_ok) vis = min(vis, i + u.g.shift + 1);
      const bool warp_on = __any_sync(0xffffffffu, vis > pc.kt0 * kTileKeys);
      const int64_t si = row_ok ? stat_index(p, u.g, h, i) : 0;
      float m = 0.f, l = 0.f;
      if (NORM != HFAN_SOFTMAX1) m = row_ok ? p.stats[si] : kPosInf;  // the threshold
      for (int j = 0; j < 2 * pc.nt; ++j, ++jj) {
        const int h2 = j & 1, kb = pc.kt0 * kTileKeys + j * kHalfKeys;
        const uint32_t s_half = s_col + h2 * kHalfKeys;
        if (ok) ok = wait_warp(&bars->s_full[q][h2], (jj >> 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (h2 == 0 && kb + kTileKeys > u.g.k_len) {
          // V rows past the sequence hold stale or foreign values: zeroed, since
          // 0 x NaN would reach O (both tiles' warps write the same zeros)
          const int item = v0 + j, vst = item % NS, lo = max(u.g.k_len - kb, 0);
          if (!(ok = wait_warp(&bars->full[vst], (item / NS) & 1, abort_flag))) break;
          uint8_t* v = smem + L::RING + vst * L::TILE;
          for (int x = r; x < (kTileKeys - lo) * 8 * NH; x += 128) {
            const int hh = x / ((kTileKeys - lo) * 8), y = x - hh * (kTileKeys - lo) * 8;
            *reinterpret_cast<uint4*>(v + hh * kHalf + lo * 128 + y * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        }
        uint32_t pk[32];
        if (warp_on) {
          uint32_t x[2][32];
          tmem_ld32(s_half, x[0]);
          tmem_ld32(s_half + 32, x[1]);
          tmem_wait_ld();
          float s[64];
#pragma unroll
          for (int e = 0; e < 64; ++e) s[e] = __uint_as_float(x[e >> 5][e & 31]);
          const int lim = vis - kb;
          if (!__all_sync(0xffffffffu, lim >= kHalfKeys)) {
#pragma unroll
            for (int e = 0; e < 64; ++e) s[e] = e < lim ? s[e] : kNegInf;
          }
          if (NORM == HFAN_SOFTMAX1) {
            float sum;
            if (!BF16 && j == 0) m = reference16(max_n<64>(s) * zs);
            for (bool again = false;; again = true) {
              const uint64_t zs2 = f2_pack(zs, zs), nm2 = f2_pack(-m, -m);
              uint64_t l2 = 0;
#pragma unroll
              for (int e = 0; e < 64; e += 2) {
                const uint64_t y = ffma2(f2_pack(s[e], s[e + 1]), zs2, nm2);
                const float e0 = ex2_ftz(f2_lo(y)), e1 = ex2_ftz(f2_hi(y));
                l2 = fadd2(l2, f2_pack(e0, e1));
                pk[e / 2] = pack2<BF16>(e0, e1);
              }
              sum = f2_lo(l2) + f2_hi(l2);
              const bool high = !(sum <= kHighSum<BF16>);
              if (again || !__any_sync(0xffffffffu, high)) break;
              // some row of the warp outgrew its reference: it moves to the
              // maximum, O and l follow, and the half is exponentiated again
              float alpha = 1.f;
              if (high) {
                const float top = max_n<64>(s) * zs, ref = fmaxf(BF16 ? top : reference16(top), m);
                alpha = exp2f(m - ref);
                m = ref;
                l *= alpha;
              }
              if (j > 0) {
                // O holds every earlier half once P V of the last one is done
                // (S of this one implies P V of the one before that)
                if (!(ok = wait_warp(&bars->pv_done[q], (jj - 1) & 1, abort_flag))) break;
                tc_fence_after();
#pragma unroll 1
                for (int cc = 0; cc < HD / 16; ++cc) {
                  uint32_t o[16];
                  tmem_ld16(o_col + cc * 16, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                  tmem_st16(o_col + cc * 16, o);
                }
              }
            }
            if (!ok) break;
            l += sum;
          } else {
            const float zl = zs * kLift<BF16, NORM>, tl = m * kLift<BF16, NORM>;
            const uint64_t zs2 = f2_pack(zl, zl), nt2 = f2_pack(-tl, -tl);
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
              const uint64_t y = ffma2(f2_pack(s[e], s[e + 1]), zs2, nt2);
              uint64_t d = f2_pack(fmaxf(f2_lo(y), 0.f), fmaxf(f2_hi(y), 0.f));
              if (NORM == HFAN_ENTMAX15) d = fmul2(d, d);
              pk[e / 2] = pack2<BF16>(f2_lo(d), f2_hi(d));
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) pk[e] = 0u;
        }
        tmem_st32(s_half, pk);
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(&bars->p_full[q][h2]);
      }
      // ---- the piece's result
      // (S of the last half implies P V of the third last: the phases of a
      // barrier are told apart by parity, so the last two are waited for in turn)
      if (ok) ok = wait_warp(&bars->pv_done[q], (jj - 2) & 1, abort_flag) && wait_warp(&bars->pv_done[q], (jj - 1) & 1, abort_flag);
      tc_fence_after();
      const int row_in_unit = q * kTileRows + r;
      const RowEnd end = end_of_row<BF16>(m, l);
      // (pieces of the sparse normalizers are whole)
      const float inv = NORM == HFAN_SOFTMAX1 ? (pc.whole ? end.inv : 1.f) : (BF16 ? 1.f : 0x1p-14f);
      T* dst = static_cast<T*>(p.o) + (int64_t)(u.g.q_start + i) * p.o_st + (int64_t)h * p.o_sh;
      float* part = ws.o + ((int64_t)pc.slot * kUnitRows + row_in_unit) * HD;
#pragma unroll 1
      for (int cc = 0; cc < HD / 32; ++cc) {
        uint32_t o[32];
        if (ok) {
          tmem_ld32(o_col + cc * 32, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0u;
        }
        if (!row_ok) continue;
        if (pc.whole) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 v;
            v.x = pack2<BF16>(__uint_as_float(o[j + 0]) * inv, __uint_as_float(o[j + 1]) * inv);
            v.y = pack2<BF16>(__uint_as_float(o[j + 2]) * inv, __uint_as_float(o[j + 3]) * inv);
            v.z = pack2<BF16>(__uint_as_float(o[j + 4]) * inv, __uint_as_float(o[j + 5]) * inv);
            v.w = pack2<BF16>(__uint_as_float(o[j + 6]) * inv, __uint_as_float(o[j + 7]) * inv);
            *reinterpret_cast<uint4*>(dst + cc * 32 + j) = v;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(part + cc * 32 + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
        }
      }
      tc_fence_before();
      warp_arrive(&bars->o_empty[q]);
      if (NORM == HFAN_SOFTMAX1 && row_ok) {
        if (pc.whole) {
          p.stats[si] = end.m;
          p.stats[(int64_t)p.hq * p.rows_total + si] = end.l;
        } else {
          ws.ml[(int64_t)pc.slot * kUnitRows + row_in_unit] = make_float2(m, l);
        }
        if (pc.kt0 == 0 && rg == 0)
          ws.info[(int64_t)(u.g.q_start + i) * p.hkv + u.kvh] = make_int4(pc.u0, u.tiles, row_in_unit, src.quota);
      }
    }
    if (!ok && lane == 0) fail(p, ctl);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// Key weights: w[key] = sum over the chunk's packed rows of p(row, key), from
// the rows' statistics.  The scores are taken transposed, S^T = K Q^T, so that
// a thread owns a key and sums over the columns without any exchange: one CTA
// takes 128 keys of one (sequence, KV head) and walks the row tiles, its two
// warpgroups alternating between them.  No reference to the maximum is
// needed: p = 2^(s zs - (m + log2 l)) (softmax1) or (s zs - tau)_+^a.
// Bound by the exponential unit (16 a cycle and SM): 2 x 512 tokens on 8k keys,
// 2.7e8 exponentials, 112 us against 63.
// ---------------------------------------------------------------------------
struct WeightBars {
  uint64_t k_full, q_full[2], q_empty[2], s_full[2], s_empty[2], drain[2];
};
template <int HD>
struct WeightLayout {
  static constexpr int NH = HD / 64;
  static constexpr uint32_t TILE = NH * kHalf;
  static constexpr uint32_t Q = TILE;
  static constexpr uint32_t CONSTS = Q + 2 * TILE;  // [2][128] row constants
  static constexpr uint32_t SUMS = CONSTS + 2 * 128 * 4;
  static constexpr uint32_t BARS = SUMS + 128 * 4;
  static constexpr uint32_t CTL = BARS + sizeof(WeightBars);
  static constexpr uint32_t TOTAL = CTL + sizeof(ChunkCtl) + 1024;
};

constexpr int kWeightThreads = 352;

template <int HD, bool BF16, int NORM>
__global__ void __launch_bounds__(kWeightThreads, 2)
    chunk_weights_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                         const AttnParams p, const ChunkPlan c, float* kw, int64_t ldw) {
  using L = WeightLayout<HD>;
  constexpr int NH = L::NH;
  allow_dependents();
  wait_for_predecessor();
  const int b = blockIdx.z, kvh = blockIdx.y, k0 = blockIdx.x * kTileKeys;
  const Geometry g = geometry(p, b);
  if (k0 >= g.k_len || g.q_len == 0) return;
  // row tiles that see the first key of this key tile
  const int i_lo = p.causal ? max(0, k0 - g.shift) : 0;
  const int t_lo = i_lo / c.tpb, t_hi = (g.q_len + c.tpb - 1) / c.tpb;
  if (t_lo >= t_hi) return;
  const int nt = t_hi - t_lo;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  WeightBars* bars = reinterpret_cast<WeightBars*>(smem + L::BARS);
  ChunkCtl* ctl = reinterpret_cast<ChunkCtl*>(smem + L::CTL);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bars->k_full, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars->q_full[s], 1);
      mbar_init(&bars->q_empty[s], 1);
      mbar_init(&bars->s_full[s], 1);
      mbar_init(&bars->s_empty[s], 4);
      mbar_init(&bars->drain[s], 1);
    }
    ctl->abort = ctl->never = 0;
    fence_barrier_init();
  }
  if (warp == 8) tmem_alloc(&ctl->tmem, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;  // S^T of warpgroup 0 | 1
  volatile int* abort_flag = &ctl->abort;
  // packed rows of row tile t, and the MMA's N (a multiple of 16) that covers them
  auto rows_of = [&](int t) { return min(c.tpb, g.q_len - t * c.tpb) * c.group; };

  if (warp == 8) {
    load_key_tile_tma<NH>(smem, &tm_k, &bars->k_full, tile_box_row(p, c, b, g.k_len, blockIdx.x), c.box_rows, kvh);
    if (lane == 0) {
      bool ok = true;
      int u = 0;
      for (; u < nt && ok; ++u) {
        const int st = u & 1;
        if (!(ok = mbar_wait(&bars->q_empty[st], ((u >> 1) & 1) ^ 1, abort_flag))) break;
        mbar_arrive_expect_tx(&bars->q_full[st], NH * c.tpb * c.group * 128);
        for (int hh = 0; hh < NH; ++hh)
          tma_load_4d(smem + L::Q + st * L::TILE + hh * kHalf, &tm_q, &bars->q_full[st], 64 * hh, kvh * c.group,
                      g.q_start + (t_lo + u) * c.tpb, 0);
      }
      if (!ok) {
        fail(p, ctl);
        mbar_wait(&bars->k_full, 0, &ctl->never);
        for (int i = max(0, u - 2); i < u; ++i) mbar_wait(&bars->q_full[i & 1], (i >> 1) & 1, &ctl->never);
      }
    }
    __syncwarp();
  } else if (warp > 8) {
    const int w = warp - 9;
    if (w < nt) {
      const uint64_t k_desc = sw128_desc(smem_u32(smem), 16, 1024);
      const uint64_t q_desc = sw128_desc(smem_u32(smem + L::Q + w * L::TILE), 16, 1024);
      bool ok = wait_warp(&bars->k_full, 0, abort_flag);
      for (int u = w; u < nt && ok; u += 2) {
        const int ph = (u >> 1) & 1;
        if (!(ok = wait_warp(&bars->q_full[w], ph, abort_flag))) break;
        if (!(ok = wait_warp(&bars->s_empty[w], ph ^ 1, abort_flag))) break;
        tc_fence_after();
        const uint32_t idesc = idesc_f16(BF16, 128, (rows_of(t_lo + u) + 15) & ~15, false, false);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t o = (kk >> 2) * kHalf + (kk & 3) * 32;
            mma_f16_ss(tmem + w * 128, desc_at(k_desc, o), desc_at(q_desc, o), idesc, kk > 0);
          }
          mma_commit(&bars->s_full[w]);
          mma_commit(&bars->q_empty[w]);
        }
        __syncwarp();
      }
      if (!ok && lane == 0) {
        fail(p, ctl);
        mma_commit(&bars->drain[w]);
        mbar_wait(&bars->drain[w], 0, &ctl->never);
      }
    }
    __syncwarp();
  } else {
    const int w = warp >> 2, r = threadIdx.x & 127;
    const uint32_t s_col = tmem + ((uint32_t)((warp & 3) * 32) << 16) + w * 128;
    float* consts = reinterpret_cast<float*>(smem + L::CONSTS) + w * 128;
    const float zs = NORM == HFAN_SOFTMAX1 ? p.scale * kLog2e : (NORM == HFAN_SPARSEMAX ? p.scale : 0.5f * p.scale);
    const uint64_t zs2 = f2_pack(zs, zs);
    const int key = k0 + r;
    float total = 0.f;
    bool ok = true;
    // statistics of this thread's row of tile t_lo + u, fetched a tile ahead
    const int rt = r / c.group, rh = kvh * c.group + r - rt * c.group;
    auto fetch = [&](int u) -> float2 {
      if (u >= nt || r >= rows_of(t_lo + u)) return make_float2(0.f, 1.f);
      const int64_t si = stat_index(p, g, rh, (t_lo + u) * c.tpb + rt);
      return make_float2(p.stats[si], NORM == HFAN_SOFTMAX1 ? p.stats[(int64_t)p.hq * p.rows_total + si] : 1.f);
    };
    float2 ahead = fetch(w);
    for (int u = w; u < nt; u += 2) {
      const int t = t_lo + u, nrows = rows_of(t);
      const float cst = NORM == HFAN_SOFTMAX1 ? -(ahead.x + log2f(ahead.y)) : -ahead.x;
      ahead = fetch(u + 2);
      named_bar_sync(1 + w, 128);  // the previous tile's constants have been read
      consts[r] = cst;
      named_bar_sync(1 + w, 128);
      if (ok) ok = wait_warp(&bars->s_full[w], (u >> 1) & 1, abort_flag);
      if (!ok) continue;  // the warpgroup keeps meeting at its barrier
      tc_fence_after();
      // rows [lo, nrows) see this thread's key
      int lo = 0;
      if (p.causal) lo = max(0, (key - g.shift - t * c.tpb)) * c.group;
      const bool full = __all_sync(0xffffffffu, lo == 0 && nrows == 128);
      uint64_t sum2 = 0;
      for (int cc = 0; cc * 32 < nrows; ++cc) {
        uint32_t x[32];
        tmem_ld32(s_col + cc * 32, x);
        tmem_wait_ld();
        const float4* c4 = reinterpret_cast<const float4*>(consts + cc * 32);
        if (!full) {
          // scores of rows that are not there may be anything
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = cc * 32 + j >= lo && cc * 32 + j < nrows ? x[j] : 0xff800000u;
        }
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 k4 = c4[j / 4];
          uint64_t a = ffma2(f2_pack(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), zs2, f2_pack(k4.x, k4.y));
          uint64_t e = ffma2(f2_pack(__uint_as_float(x[j + 2]), __uint_as_float(x[j + 3])), zs2, f2_pack(k4.z, k4.w));
          if (NORM == HFAN_SOFTMAX1) {
            a = f2_pack(ex2_ftz(f2_lo(a)), ex2_ftz(f2_hi(a)));
            e = f2_pack(ex2_ftz(f2_lo(e)), ex2_ftz(f2_hi(e)));
          } else {
            a = f2_pack(fmaxf(f2_lo(a), 0.f), fmaxf(f2_hi(a), 0.f));
            e = f2_pack(fmaxf(f2_lo(e), 0.f), fmaxf(f2_hi(e), 0.f));
            if (NORM == HFAN_ENTMAX15) {
              a = fmul2(a, a);
              e = fmul2(e, e);
            }
          }
          sum2 = fadd2(sum2, fadd2(a, e));
        }
      }
      total += f2_lo(sum2) + f2_hi(sum2);
      tc_fence_before();
      warp_arrive(&bars->s_empty[w]);
    }
    if (!ok && lane == 0) fail(p, ctl);
    float* sums = reinterpret_cast<float*>(smem + L::SUMS);
    if (w == 1) sums[r] = total;
    named_bar_sync(3, 256);
    if (w == 0 && key < g.k_len) {
      total += sums[r];
      const int64_t tok = key_token(p, g, b, key);
      if (tok >= 0) atomicAdd(kw + (int64_t)kvh * ldw + tok, total);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// ------------------------------------------------------------------ host
int pow2_divisor(int n, int most) {
  int r = 1;
  while (r < most && n % (2 * r) == 0) r *= 2;
  return r;
}

ChunkPlan plan_of(const AttnParams& p) {
  ChunkPlan c;
  c.group = p.hq / p.hkv;
  const int most = c.group < kTileRows ? kTileRows / c.group : 1;  // (larger groups run on the general kernels)
  const int longest = p.len_q < p.rows_total ? p.len_q : p.rows_total;
  c.tpb = longest < most ? (longest > 0 ? longest : 1) : most;
  c.box_rows = pow2_divisor(p.page_size, kTileKeys);
  // every sequence may leave one part-filled pair
  const int64_t pairs = p.rows_total / (2 * c.tpb) + (p.batch < p.rows_total ? p.batch : p.rows_total);
  c.pairs = (int)(pairs < 1 ? 1 : pairs);
  return c;
}

template <int HD, bool BF16, int NORM>
cudaError_t fwd_t(const AttnParams& p, const ChunkPlan& c, void* workspace, cudaStream_t s) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  CUtensorMap tq, tk, tv;
  if (!make_row_map(&tq, p, BF16, c) || !make_page_map(&tk, p.k, p.k_st, p.k_sh, p, BF16, c) ||
      !make_page_map(&tv, p.v, p.v_st, p.v_sh, p, BF16, c))
    return cudaErrorInvalidValue;
  constexpr int smem = ChunkLayout<HD>::TOTAL;
  cudaError_t e = allow_smem<chunk_fwd_kernel<HD, BF16, NORM>>(smem);
  if (e != cudaSuccess) return e;
  if (NORM == HFAN_SOFTMAX1) {
    const int ctas = sm_count();
    const PieceWs ws = piece_ws(p, ctas, kUnitRows, workspace);
    e = launch_dependent(chunk_fwd_kernel<HD, BF16, NORM>, dim3(ctas), kChunkThreads, smem, s, tq, tk, tv, p, c, ws,
                         static_cast<const int*>(nullptr));
    if (e != cudaSuccess) return e;
    return launch_dependent(combine_pieces_kernel<HD, T>, dim3(p.rows_total * p.hkv), 128, 0, s, p, ws, c.group);
  }
  int* flags = static_cast<int*>(workspace);
  e = chunk_sparse_scan(BF16 ? HFAN_BFLOAT16 : HFAN_FLOAT16, p, c, flags, s);
  if (e != cudaSuccess) return e;
  return launch_dependent(chunk_fwd_kernel<HD, BF16, NORM>, dim3(c.pairs, p.hkv), kChunkThreads, smem, s, tq, tk, tv, p, c,
                          PieceWs{}, static_cast<const int*>(flags));
}

template <int HD, bool BF16, int NORM>
cudaError_t weights_t(const AttnParams& p, const ChunkPlan& c, float* kw, int64_t ldw, cudaStream_t s) {
  CUtensorMap tq, tk;
  if (!make_row_map(&tq, p, BF16, c) || !make_page_map(&tk, p.k, p.k_st, p.k_sh, p, BF16, c))
    return cudaErrorInvalidValue;
  auto kernel = chunk_weights_kernel<HD, BF16, NORM>;
  constexpr int smem = WeightLayout<HD>::TOTAL;
  cudaError_t e = allow_smem<chunk_weights_kernel<HD, BF16, NORM>>(smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(kernel, dim3((p.len_k + kTileKeys - 1) / kTileKeys, p.hkv, p.batch), kWeightThreads, smem, s, tq, tk,
                          p, c, kw, ldw);
}

// fn<HD, BF16, NORM>(args...) for the request's types.
#define HFAN_CHUNK_DISPATCH(fn, ...)                                                                             \
  const bool bf16 = dtype == HFAN_BFLOAT16;                                                                      \
  switch (p.norm) {                                                                                              \
    case HFAN_SOFTMAX1:                                                                                          \
      return p.d == 128 ? (bf16 ? fn<128, true, HFAN_SOFTMAX1>(__VA_ARGS__) : fn<128, false, HFAN_SOFTMAX1>(__VA_ARGS__)) \
                        : (bf16 ? fn<64, true, HFAN_SOFTMAX1>(__VA_ARGS__) : fn<64, false, HFAN_SOFTMAX1>(__VA_ARGS__)); \
    case HFAN_SPARSEMAX:                                                                                         \
      return p.d == 128 ? (bf16 ? fn<128, true, HFAN_SPARSEMAX>(__VA_ARGS__) : fn<128, false, HFAN_SPARSEMAX>(__VA_ARGS__)) \
                        : (bf16 ? fn<64, true, HFAN_SPARSEMAX>(__VA_ARGS__) : fn<64, false, HFAN_SPARSEMAX>(__VA_ARGS__)); \
    default:                                                                                                     \
      return p.d == 128 ? (bf16 ? fn<128, true, HFAN_ENTMAX15>(__VA_ARGS__) : fn<128, false, HFAN_ENTMAX15>(__VA_ARGS__)) \
                        : (bf16 ? fn<64, true, HFAN_ENTMAX15>(__VA_ARGS__) : fn<64, false, HFAN_ENTMAX15>(__VA_ARGS__)); \
  }

bool keys_supported(int dtype, const AttnParams& p) {
  if (dtype != HFAN_BFLOAT16 && dtype != HFAN_FLOAT16) return false;
  if (p.d != 64 && p.d != 128) return false;
  // a swizzle atom is 8 rows of a page; masked scores are -inf before the scaling
  if (p.page_size % 8 != 0 || !(p.scale > 0.f) || p.hq / p.hkv > kTileRows) return false;
  if (p.num_cache_tokens < 1 || p.num_cache_tokens > 0x7fffffffll) return false;
  // key tiles of the whole batch are counted in 32 bits
  const ChunkPlan c = plan_of(p);
  if ((int64_t)c.pairs * p.hkv * (p.len_k / kTileKeys + 1) > 0x3fffffff) return false;
  return aligned16(p.q) && aligned16(p.k) && stride_ok(p.q_st) && stride_ok(p.q_sh) && stride_ok(p.k_st) &&
         stride_ok(p.k_sh);
}

}  // namespace

bool chunk_tc_supported(int dtype, const AttnParams& p) {
  return keys_supported(dtype, p) && aligned16(p.v) && aligned16(p.o) && stride_ok(p.v_st) &&
         stride_ok(p.v_sh) && p.o_st % 8 == 0 && p.o_sh % 8 == 0;
}

int64_t chunk_tc_workspace(const AttnParams& p, bool weights) {
  const ChunkPlan c = plan_of(p);
  if (p.norm != HFAN_SOFTMAX1) return (int64_t)c.pairs * p.hkv * 4;  // flags
  return chunk_few_applies(p, c, weights) ? chunk_few_workspace(p, c, weights) : piece_layout(p, sm_count(), kUnitRows).total;
}

static cudaError_t dense_fwd(int dtype, const AttnParams& p, const ChunkPlan& c, void* workspace, cudaStream_t s) {
  HFAN_CHUNK_DISPATCH(fwd_t, p, c, workspace, s)
}

static cudaError_t dense_weights(int dtype, const AttnParams& p, const ChunkPlan& c, float* kw, int64_t ldw, cudaStream_t s) {
  HFAN_CHUNK_DISPATCH(weights_t, p, c, kw, ldw, s)
}

cudaError_t chunk_tc_fwd(int dtype, const AttnParams& p, float* kw, int64_t ldw, void* workspace, cudaStream_t s) {
  const ChunkPlan c = plan_of(p);
  if (chunk_few_applies(p, c, kw != nullptr)) return chunk_few_fwd(dtype, p, c, kw, ldw, workspace, s);
  const cudaError_t e = dense_fwd(dtype, p, c, workspace, s);
  return e != cudaSuccess || kw == nullptr || p.len_k == 0 ? e : dense_weights(dtype, p, c, kw, ldw, s);
}

}  // namespace hfan
