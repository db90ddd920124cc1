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
// kernel (its flag tells it to), which has tau from the statistics.
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

// Raises thr to the threshold of the buffered entries alone (their sum never
// exceeds the row's) and drops the dead ones.
template <int NORM>
__device__ __noinline__ Scan compact(float* z, uint16_t* id, Scan s, int cap, float izs) {
  float t = s.thr, tau = s.thr;
  for (int it = 0; it < 8; ++it) {
    TauStats st{0.f, 0.f, 0.f, kPosInf};
    for (int e = 0; e < s.n; ++e) tau_accumulate(st, z[e * 256], t);
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
  int live = 0;
  for (int e = 0; e < s.n; ++e) {
    const float x = z[e * 256];
    if (x > s.thr) {
      id[live * 256] = id[e * 256];
      z[live++ * 256] = x;
    }
  }
  s.n = live;
  if (live > cap - 12) s.over = true;  // no room for a chunk of eight
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
        prefetch_tmap(&tm_k);
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
    if (lane == 0 && q < nact && nt > 0) {
      const uint32_t q_base = smem_u32(smem + q * L::TILE), k_base = smem_u32(smem + L::K);
      bool ok = mbar_wait(&bars->q_full, 0, abort_flag);
      int it = 0;
      for (int pass = 0; ok; ++pass) {
        for (int t = 0; t < nt; ++t, ++it) {
          const int st = it % NS, sb = it & 1;
          if (!(ok = mbar_wait(&bars->full[st], (it / NS) & 1, abort_flag))) break;
          if (!(ok = mbar_wait(&bars->s_empty[q][sb], ((it >> 1) & 1) ^ 1, abort_flag))) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t o = (kk >> 2) * kHalf + (kk & 3) * 32;
            mma_f16_ss(tmem + (2 * q + sb) * 128, sw128_desc(q_base + o, 16, 1024),
                       sw128_desc(k_base + st * L::TILE + o, 16, 1024), IDESC, kk > 0);
          }
          mma_commit(&bars->s_full[q][sb]);
          mma_commit(&bars->empty[st]);
        }
        if (!ok || !(ok = mbar_wait(&bars->ctrl, pass & 1, abort_flag))) break;
        if (!*(volatile int*)&bars->again) break;
      }
      if (!ok) {
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
    float* zb = reinterpret_cast<float*>(smem + L::Z) + slot;
    uint16_t* ib = reinterpret_cast<uint16_t*>(smem + L::ID) + slot;
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
    // 32 scores of tile t from column cc * 32, masked ones -inf
    auto load32 = [&](int t, int cc, float (&s)[32]) {
      uint32_t x[32];
      tmem_ld32(s_col + (it & 1) * 128 + cc * 32, x);
      tmem_wait_ld();
      const int lim = vis - (kt0 + t) * kTileKeys - cc * 32;
      if (__all_sync(0xffffffffu, lim >= 32)) {
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = __uint_as_float(x[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = j < lim ? __uint_as_float(x[j]) : kNegInf;
      }
    };
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
    float zmax = kNegInf;
    float tk[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
    for (int t = 0; t < nt; ++t) {
      if (!(ok = wait_s())) break;
      if (warp_on) {
        float cm[16];
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          float s[32];
          load32(t, cc, s);
#pragma unroll
          for (int e = 0; e < 4; ++e) cm[cc * 4 + e] = max_n<8>(s + e * 8);
        }
        const float tm = max_n<16>(cm);
        zmax = fmaxf(zmax, tm * zs);
        // a tile without a score above the bound changes nothing
        if (__any_sync(0xffffffffu, tm > sc.gate)) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float four[4] = {cm[4 * e], cm[4 * e + 1], cm[4 * e + 2], cm[4 * e + 3]};
            top4_merge(tk, four);
          }
          if (tk[0] > kNegInf) {
            const float zk[4] = {tk[0] * zs, tk[1] * zs, tk[2] * zs, tk[3] * zs};
            const float lb = top_bound<NORM, 4>(zk);
            if (lb > sc.thr) {
              sc.thr = lb;
              sc.gate = raw_gate(lb, izs);
            }
          }
          uint32_t mine = 0u;  // chunks of eight with a candidate
          if (!sc.over) {
#pragma unroll
            for (int e = 0; e < 16; ++e) mine |= cm[e] > sc.gate ? 1u << e : 0u;
          }
          const int lim = vis - (kt0 + t) * kTileKeys;
          for (uint32_t todo = __reduce_or_sync(0xffffffffu, mine); todo != 0u; todo &= todo - 1u) {
            const int e = __ffs(todo) - 1;
            uint32_t x[8];
            tmem_ld8(s_col + (it & 1) * 128 + e * 8, x);
            tmem_wait_ld();
            if ((mine >> e) & 1u) {
              if (sc.n > CAP - 8 && !sc.over) sc = compact<NORM>(zb, ib, sc, CAP, izs);
              if (!sc.over) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  // written at slot n, which only advances past a candidate
                  const float s = __uint_as_float(x[j]);
                  const bool in = s > sc.gate && e * 8 + j < lim;
                  if (in) {
                    zb[sc.n * 256] = s * zs;
                    ib[sc.n * 256] = (uint16_t)(t * kTileKeys + e * 8 + j);
                  }
                  sc.n += in ? 1 : 0;
                }
              }
            }
            __syncwarp();
          }
        }
      }
      free_s();
    }

    // ---- exact threshold on the union of the ranks' buffers
    float lower = kNegInf, zrow = kNegInf;
    bool over = false;
    exchange(make_float4(zmax, sc.thr, sc.over ? 1.f : 0.f, 0.f), [&](float4 v) {
      zrow = fmaxf(zrow, v.x);
      lower = fmaxf(lower, v.y);
      over |= v.z != 0.f;
    });
    auto drop = [&](float t) {
      int live = 0;
      for (int e = 0; e < sc.n; ++e) {
        const float x = zb[e * 256];
        if (x > t) {
          ib[live * 256] = ib[e * 256];
          zb[live++ * 256] = x;
        }
      }
      sc.n = live;
    };
    const bool empty = !(zrow > kNegInf);
    float tau = kPosInf, support = 0.f;
    bool pending = !empty && over;
    if (!over) {
      drop(lower);
    } else {
      sc.n = 0;
    }
    bool solving = !empty && !over;
    // (the sums are taken around the row maximum: the root depends on the support and its order alone)
    for (int step = 0; step < 64 && __any_sync(0xffffffffu, solving) && ok; ++step) {
      TauStats st{0.f, 0.f, 0.f, kPosInf}, all{0.f, 0.f, 0.f, kPosInf};
      if (solving)
        for (int e = 0; e < sc.n; ++e) tau_accumulate_ref(st, zb[e * 256], lower, zrow);
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
          for (int cc = 0; cc < 4; ++cc) {
            float s[32];
            load32(t, cc, s);
#pragma unroll
            for (int j = 0; j < 32; ++j) tau_accumulate_ref(st, s[j] * zs, lower, zrow);
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
      float* cnt = reinterpret_cast<float*>(smem + L::CNT);
      drop(tau);
      cnt[slot] = (float)sc.n;
      __syncwarp();
      if (lane < ranks) peer_arrive(&bars->lists, lane);
      ok = __all_sync(0xffffffffu, mbar_wait_cluster(&bars->lists, 0, abort_flag));
      const float* z0 = reinterpret_cast<const float*>(smem + L::Z);
      const uint16_t* i0 = reinterpret_cast<const uint16_t*>(smem + L::ID);
      // The rows of this warp, dealt to the ranks.  tau of a row is in its
      // thread's registers, so each warp serves its own 32 rows.
      const T* vbase = static_cast<const T*>(p.v) + (int64_t)kvh * p.v_sh;
      for (int rr = rank; rr < 32 && ok; rr += ranks) {
        const int rs = warp * 32 + rr;
        if (!__shfl_sync(0xffffffffu, row_ok ? 1 : 0, rr)) continue;
        const float rt = __shfl_sync(0xffffffffu, tau, rr);
        const int ri = __shfl_sync(0xffffffffu, i, rr), rh = __shfl_sync(0xffffffffu, h, rr);
        constexpr int N = HD / 32;
        float acc[N];
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = 0.f;
        for (int k = 0; k < ranks; ++k) {
          const int n = (int)(ranks == 1 ? cnt[rs] : peer_ldf(&cnt[rs], k));
          for (int e0 = 0; e0 < n; e0 += 32) {
            // lane e: probability and cache row of entry e0 + e
            float pe = 0.f;
            int64_t off = 0;
            if (e0 + lane < n) {
              const int at = (e0 + lane) * 256 + rs;
              const float d = (ranks == 1 ? z0[at] : peer_ldf(&z0[at], k)) - rt;
              const int key = k * per * kTileKeys + (int)(ranks == 1 ? i0[at] : peer_ldu16(&i0[at], k));
              const int64_t tok = key_token(p, g, b, key);
              pe = tok >= 0 ? (NORM == HFAN_SPARSEMAX ? d : d * d) : 0.f;
              off = tok >= 0 ? tok * p.v_st : 0;
            }
            const int m = min(32, n - e0);
#pragma unroll 8
            for (int e = 0; e < m; ++e) {
              const float pr = __shfl_sync(0xffffffffu, pe, e);
              const int64_t o = __shfl_sync(0xffffffffu, off, e);
              const T* v = vbase + o + lane * N;
              if constexpr (N == 4) {
                const uint2 x = __ldg(reinterpret_cast<const uint2*>(v));
                const T* xe = reinterpret_cast<const T*>(&x);
#pragma unroll
                for (int y = 0; y < 4; ++y) acc[y] = fmaf(pr, to_f32<T>(xe[y]), acc[y]);
              } else {
                const uint32_t x = __ldg(reinterpret_cast<const uint32_t*>(v));
                const T* xe = reinterpret_cast<const T*>(&x);
                acc[0] = fmaf(pr, to_f32<T>(xe[0]), acc[0]);
                acc[1] = fmaf(pr, to_f32<T>(xe[1]), acc[1]);
              }
            }
          }
        }
        T* dst = static_cast<T*>(p.o) + (int64_t)(g.q_start + ri) * p.o_st + (int64_t)rh * p.o_sh + lane * N;
        if constexpr (N == 4) {
          uint2 y;
          y.x = pack2<BF16>(acc[0], acc[1]);
          y.y = pack2<BF16>(acc[2], acc[3]);
          *reinterpret_cast<uint2*>(dst) = y;
        } else {
          *reinterpret_cast<uint32_t*>(dst) = pack2<BF16>(acc[0], acc[1]);
        }
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
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, tq, tk, p, c, ranks, flags);
}

template <int HD, bool BF16>
cudaError_t run_norm(const AttnParams& p, const ChunkPlan& c, int ranks, int* flags, cudaStream_t s) {
  return p.norm == HFAN_SPARSEMAX ? run<HD, BF16, HFAN_SPARSEMAX>(p, c, ranks, flags, s)
                                  : run<HD, BF16, HFAN_ENTMAX15>(p, c, ranks, flags, s);
}

}  // namespace

cudaError_t chunk_sparse_scan(int dtype, const AttnParams& p, const ChunkPlan& c, int* flags, cudaStream_t s) {
  // CTAs of a cluster: as many as fill the SMs, each with four key tiles or more
  const int64_t units = (int64_t)c.pairs * p.hkv, ktiles = (p.len_k + kTileKeys - 1) / kTileKeys;
  int ranks = 1;
  while (ranks < kMaxCluster && units * ranks * 2 <= sm_count() && ktiles >= ranks * 8) ranks *= 2;
  const bool bf16 = dtype == HFAN_BFLOAT16;
  if (p.d == 128) return bf16 ? run_norm<128, true>(p, c, ranks, flags, s) : run_norm<128, false>(p, c, ranks, flags, s);
  return bf16 ? run_norm<64, true>(p, c, ranks, flags, s) : run_norm<64, false>(p, c, ranks, flags, s);
}

}  // namespace hfan
