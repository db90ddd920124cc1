// sparsemax / entmax15 attention of a ragged chunk over a paged cache (tcgen05;
// the requests of paged_chunk_tc.cu).
//
// The threshold tau of a row is needed before any probability is known.  One
// CTA scans the keys of two tiles of 128 packed rows (S = Q K^T only; row
// thread = TMEM lane, which reads its whole S row) and every row buffers, in
// shared memory, the scores above a rising lower bound of tau with their keys.
// The bound comes from the four largest 8-key maxima and, when the buffer is
// full, from the threshold of what it holds; it never exceeds tau, so the exact
// tau of the row is solved on the buffer (common.cuh).  What is left above tau
// is the row's whole support, a few keys: P V is gathered from their V rows,
// and no second pass over the keys takes place.
//
// Rows with more live candidates than the buffer holds are solved by bracket
// sweeps over all keys; a CTA with such a row leaves its P V to the dense
// kernel (its flag tells it to), which has tau from the statistics.  That is a
// matter of the scores: entmax15, 4 x 256 tokens on 8k keys, takes 223 us with
// queries of twice unit deviation (supports of 8-10 keys), 260 at 1.5 and 862 at
// unit deviation (about 25 keys, and nearly every unit has a row over the
// buffer); sparsemax 139, 146 and 158.
//
// Measured: sparsemax, 4 x up to 256 tokens on up to 8k keys: 85 us, of a CTA's
// 118k cycles 73k in the scan, 9k in the threshold, 29k in the gather.  The scan
// is bound by its row warps: three of four groups of 32 columns have a candidate
// for one of a warp's 32 rows (3.0k cycles a key tile, the products need 1.0k).
// A separate pass for the maxima, so that the second one buffers little, took as
// long as it saved.
//
// With few rows a cluster of up to 8 CTAs shares a tile pair, each scanning a
// part of the keys: the rows' sums are exchanged through distributed shared
// memory in rank order, so that every rank takes the same steps, and the
// gather is dealt out by rows.
#include <cuda.h>

#include "common.cuh"
#include "paged_chunk.cuh"
#include "paged_serving.cuh"
#include "params.cuh"
#include "tc_common.cuh"
#include "tc_ptx.cuh"
#include "tc_sparse.cuh"

namespace hfan {
namespace {

using namespace tc;

constexpr int kThreads = 384;  // 8 row warps, producer, two issuers, one that fills the warpgroup
constexpr int kMaxStages = 4;
constexpr int kMaxSweeps = 48;
constexpr int kMaxCluster = 8;
constexpr int kMaxIdTiles = 512;  // key tiles of one CTA whose keys fit 16-bit ids

template <int HD>
struct SparseLayout {
  static constexpr int NH = HD / 64;
  static constexpr int STAGES = HD == 128 ? 2 : 4;
  static constexpr int CAP = HD == 128 ? 56 : 80;  // buffered candidates of a row
  static constexpr uint32_t TILE = NH * kHalf;
  static constexpr uint32_t K = 2 * TILE;
  static constexpr uint32_t Z = K + STAGES * TILE;        // float [CAP][256]
  static constexpr uint32_t ID = Z + CAP * 256 * 4;       // uint16 [CAP][256]
  static constexpr uint32_t XCH = ID + CAP * 256 * 2;     // float4 [2][256]
  static_assert(CAP * 256 * 4 <= (2 + STAGES) * NH * kHalf, "the rows of the support go over the Q and K tiles");
  static constexpr uint32_t CNT = XCH + 2 * 256 * 16;     // float [256] entries left above tau
  static constexpr uint32_t BARS = CNT + 256 * 4;
  static constexpr uint32_t TOTAL = BARS + 512 + 1024;
};

struct SparseBars {
  uint64_t q_full, full[kMaxStages], empty[kMaxStages];
  uint64_t s_full[2][2], s_empty[2][2], ctrl, drain[2];
  uint64_t xch[8][2];  // one pair per row warp: its counterparts of the cluster
  uint64_t lists;      // every row warp of the cluster
  uint32_t tmem;
  int abort, never, again;
};
static_assert(sizeof(SparseBars) <= 512, "SparseBars outgrew its place");

__device__ __forceinline__ void fail(const AttnParams& p, SparseBars* s) {
  s->abort = 1;
  if (p.dev_status) atomicCAS(p.dev_status, kDevOk, kDevWaitTimeout);
}

struct Scan {
  int n;       // buffered entries, in key order (some may be at or below thr)
  bool over;   // more live candidates than the buffer holds
  float thr;   // lower bound of tau, z units
  float gate;  // the same in raw scores, or slightly below
};

// Raises thr towards the threshold of the buffered entries alone (their sum
// never exceeds the row's, and the steps never overshoot) and drops the dead.
// z, id: shared-space addresses of the row's columns, entries kZStep and
// kIdStep bytes apart.
constexpr uint32_t kZStep = 256 * 4, kIdStep = 256 * 2;

__device__ __forceinline__ int drop_dead(uint32_t z, uint32_t id, int n, float t) {
  int live = 0;
#pragma unroll 4
  for (int e = 0; e < n; ++e) {
    const float x = lds_f32(z + e * kZStep);
    const uint32_t k = lds_u16(id + e * kIdStep);
    const bool in = x > t;
    sts_f32_if(in, z + live * kZStep, x);
    sts_u16_if(in, id + live * kIdStep, k);
    live += in ? 1 : 0;
  }
  return live;
}

template <int NORM>
__device__ __noinline__ Scan compact(uint32_t z, uint32_t id, Scan s, int cap, float izs) {
  if (s.over) return s;
  float t = s.thr, tau = s.thr;
#pragma unroll 1
  for (int it = 0; it < 3; ++it) {
    TauStats st{0.f, 0.f, 0.f, kPosInf};
#pragma unroll 4
    for (int e = 0; e < s.n; ++e) tau_accumulate(st, lds_f32(z + e * kZStep), t);
    if (st.cnt == 0.f) break;
    if (tau_step(NORM, st, &t, &tau)) {
      t = tau;
      break;
    }
  }
  if (t > s.thr) {
    s.thr = t;
    s.gate = raw_gate(t, izs);
  }
  s.n = drop_dead(z, id, s.n, s.thr);
  if (s.n > cap - 12) s.over = true;  // hardly any room left
  return s;
}

template <int HD, bool BF16, int NORM>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_sparse_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const AttnParams p, const ChunkPlan c, int ranks, int* flags) {
  using L = SparseLayout<HD>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  constexpr int NH = L::NH, NS = L::STAGES, CAP = L::CAP;
  constexpr uint32_t IDESC = idesc_f16(BF16, 128, 128, false, false);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  SparseBars* bars = reinterpret_cast<SparseBars*>(smem + L::BARS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = ranks > 1 ? (int)cluster_rank() : 0;

  allow_dependents();
  if (warp == 8 && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
  }
  wait_for_predecessor();
  const UnownedRows rest(p);
  for (int x = blockIdx.x; x < rest.count; x += gridDim.x)
    store_empty_rows<T, uint4>(p, rest.at(x), blockIdx.y * c.group, c.group);
  if (warp == 11 && blockIdx.x == 0 && blockIdx.y == 0) record_bad_offsets(p, lane, 32);
  int b, pair;
  const int unit = blockIdx.x / ranks;
  if (!find_group(p, 2 * c.tpb, unit, &b, &pair)) return;  // the whole cluster alike
  const Geometry g = geometry(p, b);
  const int kvh = blockIdx.y;
  const int tok0 = pair * 2 * c.tpb, ntok = min(2 * c.tpb, g.q_len - tok0);
  const int nact = ntok > c.tpb ? 2 : 1;
  const int k_hi = p.causal ? min(g.k_len, tok0 + ntok + g.shift) : g.k_len;
  const int n_all = k_hi > 0 ? (k_hi + kTileKeys - 1) / kTileKeys : 0;
  const int per = (n_all + ranks - 1) / ranks, kt0 = rank * per, nt = max(0, min(per, n_all - kt0));
  const int row_threads = 128 * nact;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->ctrl, 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], nact);
    }
    for (int q = 0; q < 2; ++q) {
      mbar_init(&bars->drain[q], 1);
      for (int s = 0; s < 2; ++s) {
        mbar_init(&bars->s_full[q][s], 1);
        mbar_init(&bars->s_empty[q][s], 4);
      }
    }
    for (int w = 0; w < 8; ++w)
      for (int s = 0; s < 2; ++s) mbar_init(&bars->xch[w][s], ranks);
    mbar_init(&bars->lists, ranks * nact * 4);
    bars->abort = bars->never = bars->again = 0;
    fence_barrier_init();
  }
  if (warp == 8) tmem_alloc(&bars->tmem, 512);
  tc_fence_before();
  __syncthreads();
  if (ranks > 1) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;  // S of (tile q, buffer s) at column (2 q + s) 128
  volatile int* abort_flag = &bars->abort;

  if (warp == 8) {
    // ------------------------------------------------------------ producer
    if (nt > 0) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars->q_full, nact * NH * c.tpb * c.group * 128);
        for (int q = 0; q < nact; ++q)
          for (int hh = 0; hh < NH; ++hh)
            tma_load_4d(smem + q * L::TILE + hh * kHalf, &tm_q, &bars->q_full, 64 * hh, kvh * c.group,
                        g.q_start + tok0 + q * c.tpb, 0);
      }
      bool ok = true;
      int issued = 0;
      for (int pass = 0; ok; ++pass) {
        int row = tile_box_row(p, c, b, g.k_len, kt0);
        for (int t = 0; t < nt; ++t) {
          const int next = t + 1 < nt ? tile_box_row(p, c, b, g.k_len, kt0 + t + 1) : -1;
          const int st = issued % NS;
          if (!(ok = wait_warp(&bars->empty[st], ((issued / NS) & 1) ^ 1, abort_flag))) break;
          load_key_tile_tma<NH>(smem + L::K + st * L::TILE, &tm_k, &bars->full[st], row, c.box_rows, kvh);
          ++issued;
          row = next;
        }
        if (!ok || !(ok = wait_warp(&bars->ctrl, pass & 1, abort_flag))) break;
        if (!*(volatile int*)&bars->again) break;
      }
      if (!ok && lane == 0) {
        fail(p, bars);
        mbar_wait(&bars->q_full, 0, &bars->never);
        for (int i = max(0, issued - NS); i < issued; ++i) mbar_wait(&bars->full[i % NS], (i / NS) & 1, &bars->never);
      }
    }
    __syncwarp();
  } else if (warp > 8) {
    // ------------------------------------------------------------ MMA issuers
    const int q = warp - 9;
    if (q < nact && nt > 0) {
      const uint64_t q_desc = sw128_desc(smem_u32(smem + q * L::TILE), 16, 1024);
      const uint32_t k_base = smem_u32(smem + L::K);
      bool ok = wait_warp(&bars->q_full, 0, abort_flag);
      int it = 0;
      for (int pass = 0; ok; ++pass) {
        for (int t = 0; t < nt; ++t, ++it) {
          const int st = it % NS, sb = it & 1;
          if (!(ok = wait_warp(&bars->full[st], (it / NS) & 1, abort_flag))) break;
          if (!(ok = wait_warp(&bars->s_empty[q][sb], ((it >> 1) & 1) ^ 1, abort_flag))) break;
          tc_fence_after();
          const uint64_t k_desc = sw128_desc(k_base + st * L::TILE, 16, 1024);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
              const uint32_t o = (kk >> 2) * kHalf + (kk & 3) * 32;
              mma_f16_ss(tmem + (2 * q + sb) * 128, desc_at(q_desc, o), desc_at(k_desc, o), IDESC, kk > 0);
            }
            mma_commit(&bars->s_full[q][sb]);
            mma_commit(&bars->empty[st]);
          }
          __syncwarp();
        }
        if (!ok || !(ok = wait_warp(&bars->ctrl, pass & 1, abort_flag))) break;
        if (!*(volatile int*)&bars->again) break;
      }
      if (!ok && lane == 0) {
        fail(p, bars);
        mma_commit(&bars->drain[q]);
        mbar_wait(&bars->drain[q], 0, &bars->never);
      }
    }
    __syncwarp();
  } else if ((warp >> 2) < nact) {
    // ------------------------------------------------------------ row warps
    const int q = warp >> 2, r = threadIdx.x & 127, slot = threadIdx.x;  // slot: 128 q + r
    const int i = tok0 + q * c.tpb + r / c.group;
    const bool row_ok = r < c.tpb * c.group && i < g.q_len;
    const int h = kvh * c.group + r % c.group;
    const uint32_t s_col = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 2 * q * 128;
    int vis = row_ok ? g.k_len : 0;
    if (p.causal && row_ok) vis = min(vis, i + g.shift + 1);
    const bool warp_on = __any_sync(0xffffffffu, vis > kt0 * kTileKeys);
    const float zs = NORM == HFAN_SPARSEMAX ? p.scale : 0.5f * p.scale, izs = 1.f / zs;
    const uint32_t zb = smem_u32(smem + L::Z) + slot * 4, ib = smem_u32(smem + L::ID) + slot * 2;
    float4* xch = reinterpret_cast<float4*>(smem + L::XCH);
    bool ok = true;
    int it = 0, rounds = 0;

    auto wait_s = [&]() -> bool {
      if (!wait_warp(&bars->s_full[q][it & 1], (it >> 1) & 1, abort_flag)) return false;
      tc_fence_after();
      return true;
    };
    auto free_s = [&]() {
      tc_fence_before();
      warp_arrive(&bars->s_empty[q][it & 1]);
      ++it;
    };
    // scores of columns [32 cc, 32 cc + 32) of tile t, masked ones -inf
    auto mask32 = [&](int t, int cc, uint32_t (&x)[32]) {
      const int lim = vis - (kt0 + t) * kTileKeys - cc * 32;
      if (!__all_sync(0xffffffffu, lim >= 32)) {
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = j < lim ? x[j] : 0xff800000u;
      }
    };
    auto s_at = [&](int cc) { return s_col + (it & 1) * 128 + cc * 32; };
    // Publishes v and visits every rank's value of the same row in rank order.
    // Two buffers suffice: a warp writes one again only after its counterparts
    // arrived for the other, which they do when they have read this one.
    auto exchange = [&](float4 v, auto&& visit) {
      if (ranks == 1) {
        visit(v);
        return;
      }
      const int par = rounds & 1;
      xch[par * 256 + slot] = v;
      __syncwarp();
      if (lane < ranks) peer_arrive(&bars->xch[warp][par], lane);
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait_cluster(&bars->xch[warp][par], (rounds >> 1) & 1, abort_flag));
      if (ok)
        for (int k = 0; k < ranks; ++k) visit(peer_ld4(&xch[par * 256 + slot], k));
      ++rounds;
    };

    // ---- scan
    Scan sc{0, false, kNegInf, kNegInf};
    float smax = kNegInf;
    float tk[4] = {kNegInf, kNegInf, kNegInf, kNegInf};  // the largest 8-key maxima
    auto raise = [&]() {
      if (tk[0] > kNegInf) {
        const float zk[4] = {tk[0] * zs, tk[1] * zs, tk[2] * zs, tk[3] * zs};
        const float lb = top_bound<NORM, 4>(zk);
        if (lb > sc.thr) {
          sc.thr = lb;
          sc.gate = raw_gate(lb, izs);
        }
      }
    };
    for (int t = 0; t < nt; ++t) {
      if (!(ok = wait_s())) break;
      if (warp_on) {
        if (t == 0) {
          // the first tile's maxima give a bound before anything is buffered
#pragma unroll 1
          for (int cc = 0; cc < 4; ++cc) {
            uint32_t x[32];
            tmem_ld32(s_at(cc), x);
            tmem_wait_ld();
            mask32(t, cc, x);
            const float* s = reinterpret_cast<const float*>(x);
            const float cm[4] = {max_n<8>(s), max_n<8>(s + 8), max_n<8>(s + 16), max_n<8>(s + 24)};
            top4_merge(tk, cm);
          }
          raise();
          tk[0] = tk[1] = tk[2] = tk[3] = kNegInf;  // (merged again below)
        }
        bool heavy = false;
#pragma unroll 1  // (unrolled, the code of a tile outgrows the instruction caches)
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t x[32];
          tmem_ld32(s_at(cc), x);
          tmem_wait_ld();
          mask32(t, cc, x);
          const float* s = reinterpret_cast<const float*>(x);
          float hm[8], cm[4];  // maxima of four and of eight keys
#pragma unroll
          for (int e = 0; e < 8; ++e) hm[e] = max_n<4>(s + 4 * e);
#pragma unroll
          for (int e = 0; e < 4; ++e) cm[e] = fmaxf(hm[2 * e], hm[2 * e + 1]);
          const float gm = fmaxf(max3f(cm[0], cm[1], cm[2]), cm[3]);
          smax = fmaxf(smax, gm);
          // keys at or below the bound change nothing: no candidate, and no
          // set of them has a threshold above it
          if (__any_sync(0xffffffffu, gm > sc.gate)) {
            heavy = true;
            top4_merge(tk, cm);
            const bool tight = __any_sync(0xffffffffu, sc.n > CAP - 32 && !sc.over);  // (the group may fill a buffer)
            const uint32_t id0 = t * kTileKeys + cc * 32;
            uint32_t za = zb + sc.n * kZStep, ia = ib + sc.n * kIdStep;
            float gate = sc.over ? kPosInf : sc.gate;
            // Few lanes have a candidate, and those one or two: every lane takes
            // the quarters of eight it has, one per turn, brings its four scores
            // to the front by selections and pushes them predicated.  (Divergent
            // branches took several times as long, 32 predicated pushes twice.)
            uint32_t mine = 0u;
#pragma unroll
            for (int e = 0; e < 8; ++e) mine |= hm[e] > gate ? 1u << e : 0u;
            while (__any_sync(0xffffffffu, mine != 0u)) {
              // All lanes compact when one has to: they do it in the same time,
              // and their raised bounds keep them from having to one by one.
              if (tight) {
                sc.n = (za - zb) / kZStep;
                if (__any_sync(0xffffffffu, sc.n > CAP - 4 && !sc.over)) {
                  sc = compact<NORM>(zb, ib, sc, CAP, izs);
                  za = zb + sc.n * kZStep;
                  ia = ib + sc.n * kIdStep;
                  gate = sc.over ? kPosInf : sc.gate;
                }
              }
              const int e = mine != 0u ? __ffs(mine) - 1 : 0;
              const float lim_e = mine != 0u ? gate : kPosInf;
              mine &= mine - 1u;
              const bool b0 = e & 1, b1 = e & 2, b2 = e & 4;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float v0 = b0 ? s[4 + k] : s[k], v1 = b0 ? s[12 + k] : s[8 + k];
                const float v2 = b0 ? s[20 + k] : s[16 + k], v3 = b0 ? s[28 + k] : s[24 + k];
                const float x = b2 ? (b1 ? v3 : v2) : (b1 ? v1 : v0);
                push_if_above(x, lim_e, x * zs, id0 + 4 * e + k, za, ia, kZStep, kIdStep);
              }
            }
            sc.n = (za - zb) / kZStep;
          }
        }
        if (heavy) raise();
      }
      free_s();
    }
    const float zmax = smax * zs;

    // ---- exact threshold on the union of the ranks' buffers
    float lower = kNegInf, zrow = kNegInf;
    bool over = false;
    exchange(make_float4(zmax, sc.thr, sc.over ? 1.f : 0.f, 0.f), [&](float4 v) {
      zrow = fmaxf(zrow, v.x);
      lower = fmaxf(lower, v.y);
      over |= v.z != 0.f;
    });
    const bool empty = !(zrow > kNegInf);
    float tau = kPosInf, support = 0.f;
    bool pending = !empty && over;
    if (!over) {
      sc.n = drop_dead(zb, ib, sc.n, lower);
    } else {
      sc.n = 0;
    }
    bool solving = !empty && !over;
    // (the sums are taken around the row maximum: the root depends on the support and its order alone)
    for (int step = 0; step < 64 && __any_sync(0xffffffffu, solving) && ok; ++step) {
      TauStats st{0.f, 0.f, 0.f, kPosInf}, all{0.f, 0.f, 0.f, kPosInf};
      if (solving)
#pragma unroll 4
        for (int e = 0; e < sc.n; ++e) tau_accumulate_ref(st, lds_f32(zb + e * kZStep), lower, zrow);
      exchange(make_float4(st.cnt, st.s1, st.s2, st.zmin), [&](float4 v) {
        all.cnt += v.x;
        all.s1 += v.y;
        all.s2 += v.z;
        all.zmin = fminf(all.zmin, v.w);
      });
      if (solving) {
        support = all.cnt;
        if (all.cnt == 0.f) {
          solving = false;
          pending = over = true;
        } else if (tau_step_ref(NORM, all, zrow, &lower, &tau)) {
          solving = false;
        }
      }
    }
    if (solving) {
      pending = over = true;
      tau = kPosInf;
    }

    // ---- rows that outgrew the buffer: bracket sweeps over all keys
    for (int sweep = 0;; ++sweep) {
      const bool again = named_bar_or(1, row_threads, pending) && sweep < kMaxSweeps && *abort_flag == 0;
      const bool go = named_bar_or(1, row_threads, again);  // one answer for the block
      if (threadIdx.x == 0) {
        bars->again = go ? 1 : 0;
        mbar_arrive(&bars->ctrl);
      }
      if (!go) break;
      TauStats st{0.f, 0.f, 0.f, kPosInf}, all{0.f, 0.f, 0.f, kPosInf};
      for (int t = 0; t < nt && ok; ++t) {
        if (!(ok = wait_s())) break;
        if (__any_sync(0xffffffffu, pending)) {
#pragma unroll 1
          for (int cc = 0; cc < 4; ++cc) {
            uint32_t x[32];
            tmem_ld32(s_at(cc), x);
            tmem_wait_ld();
            mask32(t, cc, x);
#pragma unroll
            for (int j = 0; j < 32; ++j) tau_accumulate_ref(st, __uint_as_float(x[j]) * zs, lower, zrow);
          }
        }
        free_s();
      }
      exchange(make_float4(st.cnt, st.s1, st.s2, st.zmin), [&](float4 v) {
        all.cnt += v.x;
        all.s1 += v.y;
        all.s2 += v.z;
        all.zmin = fminf(all.zmin, v.w);
      });
      if (pending && ok) {
        support = all.cnt;
        pending = !tau_step_ref(NORM, all, zrow, &lower, &tau);
      }
    }
    if (!ok && lane == 0) fail(p, bars);
    if (row_ok && rank == 0) {
      const int64_t si = stat_index(p, g, h, i);
      p.stats[si] = empty ? kPosInf : tau;
      p.stats[(int64_t)p.hq * p.rows_total + si] = support;
    }

    // ---- P V from the buffered support
    const bool dense = named_bar_or(1, row_threads, over || !ok) || per > kMaxIdTiles;
    if (threadIdx.x == 0 && rank == 0) flags[unit * p.hkv + kvh] = dense ? 1 : 0;
    if (!dense) {
      // Every thread leaves its support in place as (p, cache row); the rows
      // go over the Q and K tiles, which nothing reads any more.
      float* cnt = reinterpret_cast<float*>(smem + L::CNT);
      int* rows = reinterpret_cast<int*>(smem);  // [CAP][256]
      int live = 0;
#pragma unroll 4
      for (int e = 0; e < sc.n; ++e) {
        const float d = lds_f32(zb + e * kZStep) - tau;
        const uint32_t k = lds_u16(ib + e * kIdStep);
        const bool in = d > 0.f;
        sts_f32_if(in, zb + live * kZStep, NORM == HFAN_SPARSEMAX ? d : d * d);
        sts_u16_if(in, ib + live * kIdStep, k);
        live += in ? 1 : 0;
      }
#pragma unroll 4
      for (int e = 0; e < live; ++e) {
        const int64_t tok = key_token(p, g, b, kt0 * kTileKeys + (int)lds_u16(ib + e * kIdStep));
        sts_f32_if(tok < 0, zb + e * kZStep, 0.f);  // (a page id outside the cache: its V reads as zeros)
        rows[e * 256 + slot] = max((int)tok, 0);
      }
      cnt[slot] = (float)live;
      __syncwarp();
      if (lane < ranks) peer_arrive(&bars->lists, lane);
      if (!mbar_wait_cluster(&bars->lists, 0, abort_flag)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      // Groups of eight lanes take a row each (16 head dims of a lane at HD =
      // 128), four rows of the warp at a time; the ranks share the rows.
      constexpr int N = HD / 8, V = N / 8;  // values and 16-byte loads of a lane
      const float* z0 = reinterpret_cast<const float*>(smem + L::Z);
      const T* vbase = static_cast<const T*>(p.v) + (int64_t)kvh * p.v_sh + (lane & 7) * N;
      for (int r0 = rank * 4; r0 < 32 && ok; r0 += ranks * 4) {
        const int rr = r0 + (lane >> 3), rs = warp * 32 + rr;
        const bool on = __shfl_sync(0xffffffffu, row_ok ? 1 : 0, rr) != 0;
        const int ri = __shfl_sync(0xffffffffu, i, rr), rh = __shfl_sync(0xffffffffu, h, rr);
        uint64_t acc[N / 2];
#pragma unroll
        for (int e = 0; e < N / 2; ++e) acc[e] = 0ull;
        for (int k = 0; on && k < ranks; ++k) {
          const int n = (int)(ranks == 1 ? cnt[rs] : peer_ldf(&cnt[rs], k));
#pragma unroll 4
          for (int e = 0; e < n; ++e) {
            float pr;
            int row;
            if (ranks == 1) {
              pr = z0[e * 256 + rs];
              row = rows[e * 256 + rs];
            } else {
              pr = peer_ldf(&z0[e * 256 + rs], k);
              row = __float_as_int(peer_ldf(reinterpret_cast<const float*>(&rows[e * 256 + rs]), k));
            }
            const uint4* v = reinterpret_cast<const uint4*>(vbase + (int64_t)row * p.v_st);
            const uint64_t p2 = f2_pack(pr, pr);
            uint4 x[V];
#pragma unroll
            for (int y = 0; y < V; ++y) x[y] = v[y];  // (coherent: an append or eviction may end during this launch)
#pragma unroll
            for (int y = 0; y < V; ++y) {
              acc[4 * y + 0] = ffma2(p2, unpack2<BF16>(x[y].x), acc[4 * y + 0]);
              acc[4 * y + 1] = ffma2(p2, unpack2<BF16>(x[y].y), acc[4 * y + 1]);
              acc[4 * y + 2] = ffma2(p2, unpack2<BF16>(x[y].z), acc[4 * y + 2]);
              acc[4 * y + 3] = ffma2(p2, unpack2<BF16>(x[y].w), acc[4 * y + 3]);
            }
          }
        }
        if (on) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.o) + (int64_t)(g.q_start + ri) * p.o_st +
                                                (int64_t)rh * p.o_sh + (lane & 7) * N);
#pragma unroll
          for (int y = 0; y < V; ++y)
            dst[y] = make_uint4(pack2<BF16>(f2_lo(acc[4 * y]), f2_hi(acc[4 * y])),
                                pack2<BF16>(f2_lo(acc[4 * y + 1]), f2_hi(acc[4 * y + 1])),
                                pack2<BF16>(f2_lo(acc[4 * y + 2]), f2_hi(acc[4 * y + 2])),
                                pack2<BF16>(f2_lo(acc[4 * y + 3]), f2_hi(acc[4 * y + 3])));
        }
        __syncwarp();
      }
      if (!ok && lane == 0) fail(p, bars);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (ranks > 1) cluster_sync();  // the peers have read this CTA's lists
}

template <int HD, bool BF16, int NORM>
cudaError_t run(const AttnParams& p, const ChunkPlan& c, int ranks, int* flags, cudaStream_t s) {
  CUtensorMap tq, tk;
  if (!make_row_map(&tq, p, BF16, c) || !make_page_map(&tk, p.k, p.k_st, p.k_sh, p, BF16, c))
    return cudaErrorInvalidValue;
  auto kernel = chunk_sparse_kernel<HD, BF16, NORM>;
  constexpr int smem = SparseLayout<HD>::TOTAL;
  cudaError_t e = allow_smem<chunk_sparse_kernel<HD, BF16, NORM>>(smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(c.pairs * ranks, p.hkv, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ranks > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, tq, tk, p, c, ranks, flags);
}

template <int HD, bool BF16>
cudaError_t run_norm(const AttnParams& p, const ChunkPlan& c, int ranks, int* flags, cudaStream_t s) {
  return p.norm == HFAN_SPARSEMAX ? run<HD, BF16, HFAN_SPARSEMAX>(p, c, ranks, flags, s)
                                  : run<HD, BF16, HFAN_ENTMAX15>(p, c, ranks, flags, s);
}

}  // namespace

cudaError_t chunk_sparse_scan(int dtype, const AttnParams& p, const ChunkPlan& c, int* flags, cudaStream_t s) {
  // CTAs of a cluster: up to two waves over the SMs (the bound counts pairs
  // that ragged sequences do not fill), each CTA with four key tiles or more.
  // Measured with 1 / 2 / 4 / 8 ranks (sparsemax, 8 KV heads, us; entmax15 alike):
  // 1 token on 32k keys 266 / 153 / 96 / 69 (the rule: 8), 4 x 1 on 2k 42 / 37 /
  // 34 / 72 (4), 8 x 1 on 8k 92 / 67 / 92 / 170 (2), 4 x 256 on 8k 140 / 179 /
  // 240 / 419 (1).  A bound that is not reached costs: 2 x 130 tokens on 3k take
  // 83 / 63 / 87 / 129, and the rule says 4.
  const int64_t units = (int64_t)c.pairs * p.hkv, ktiles = (p.len_k + kTileKeys - 1) / kTileKeys;
  int ranks = 1;
  while (ranks < kMaxCluster && units * ranks <= sm_count() && ktiles >= ranks * 8) ranks *= 2;
  const bool bf16 = dtype == HFAN_BFLOAT16;
  if (p.d == 128) return bf16 ? run_norm<128, true>(p, c, ranks, flags, s) : run_norm<128, false>(p, c, ranks, flags, s);
  return bf16 ? run_norm<64, true>(p, c, ranks, flags, s) : run_norm<64, false>(p, c, ranks, flags, s);
}

}  // namespace hfan
