// How the tensor-core chunk kernels share the work of a ragged batch.
//
// A unit is a group of `per` tokens of one sequence under one KV head; its work
// is its key tiles.  All units' tiles, in (sequence, KV head, group) order,
// form one line that is cut into equal stretches, one per CTA: every SM gets
// the same number of tiles however ragged the lengths are.  A stretch may start
// and end inside a unit, so a CTA has at most two partial results, its first
// piece and its last; combine_pieces_kernel joins the pieces of a unit.
#pragma once

#include "paged_chunk.cuh"
#include "tc_ptx.cuh"

namespace hfan {

// What the pieces of a unit leave for combine_pieces_kernel.
struct PieceWs {
  float* o;    // [2 * ctas][rows of a unit][D] unscaled O of a partial piece
  float2* ml;  // [2 * ctas][rows of a unit] (reference m, sum l)
  int4* info;  // [total_q][hkv] (first tile of the unit on the line, its tiles, first row of the token, tiles of a CTA)
  int rows;    // rows of a unit
  int ctas;
};

struct Unit {
  int b, kvh, tok0, ntok;  // tokens [tok0, tok0 + ntok) of sequence b
  int tiles;               // key tiles it sees (at least one, which may be masked altogether)
  Geometry g;
};

struct Piece {
  int kt0, nt;  // key tiles [kt0, kt0 + nt) of the unit
  int u0;       // the unit's first tile on the line
  int slot;     // partial results
  bool whole;
};

class Walk {
 public:
  Unit u;
  Piece piece;
  int quota;  // tiles of a CTA

  // Whole-warp call: finds the start of this CTA's stretch.
  __device__ __forceinline__ Walk(const AttnParams& p, int per) : p_(p), per_(per) {
    const int lane = threadIdx.x & 31;
    int total = 0, w0 = 0;
    for (int base = 0; base < p.batch; base += 32) {
      const int w = base + lane < p.batch ? sequence_tiles(base + lane) * p.hkv : 0;
      if (base == 0) w0 = w;
      total += __reduce_add_sync(0xffffffffu, w);
    }
    quota = max((total + (int)gridDim.x - 1) / (int)gridDim.x, 2);
    at_ = (int)blockIdx.x * quota;
    const int end = min(at_ + quota, total);
    end_ = at_;
    if (at_ >= end) return;
    int before = 0;
    for (int base = 0; base < p.batch; base += 32) {
      const int w = base == 0 ? w0 : (base + lane < p.batch ? sequence_tiles(base + lane) * p.hkv : 0);
      int inc = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + inc > at_);
      if (hit) {
        const int l = __ffs(hit) - 1;
        enter(base + l);
        int off = max(at_ - before - __shfl_sync(0xffffffffu, inc - w, l), 0);
        const int one = __shfl_sync(0xffffffffu, w, l) / p.hkv;
        u.kvh = min(off / one, p.hkv - 1);
        off -= u.kvh * one;
        group_ = 0;
        load_group();
        while (off >= u.tiles && (group_ + 1) * per_ < u.g.q_len) {
          off -= u.tiles;
          ++group_;
          load_group();
        }
        u0_ = at_ - off;
        end_ = end;
        break;
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
  }

  // Moves to the next piece of the stretch; false when it is done.
  __device__ __forceinline__ bool next() {
    if (at_ >= end_) return false;
    if (at_ >= u0_ + u.tiles) {  // the next unit
      u0_ = at_;
      ++group_;
      if (group_ * per_ >= u.g.q_len) {
        group_ = 0;
        if (++u.kvh == p_.hkv) {
          u.kvh = 0;
          int b = u.b, s;
          do ++b;  // (the line has tiles left, so some sequence follows)
          while (b + 1 < p_.batch && chunk_tokens(p_, b, &s) == 0);
          enter(b);
        }
      }
      load_group();
    }
    piece.kt0 = at_ - u0_;
    piece.nt = min(u.tiles - piece.kt0, end_ - at_);
    piece.u0 = u0_;
    piece.whole = piece.nt == u.tiles;
    piece.slot = 2 * (int)blockIdx.x + (at_ == (int)blockIdx.x * quota ? 0 : 1);
    at_ += piece.nt;
    return true;
  }

 private:
  __device__ __forceinline__ int group_tiles(int n, int k_len, int j) const {
    const int end = min((j + 1) * per_, n);  // tokens up to here see keys up to end + (k_len - n)
    const int k_hi = p_.causal ? min(k_len, end + k_len - n) : k_len;
    return max((k_hi + kTileKeys - 1) / kTileKeys, 1);
  }
  __device__ __forceinline__ int sequence_tiles(int b) const {
    int s;
    const int n = chunk_tokens(p_, b, &s);
    const int k_len = min(max(p_.seq_lens[b], 0), p_.len_k);
    int sum = 0;
    for (int j = 0; j * per_ < n; ++j) sum += group_tiles(n, k_len, j);
    return sum;
  }
  __device__ __forceinline__ void enter(int b) {
    u.b = b;
    u.g = geometry(p_, b);
  }
  __device__ __forceinline__ void load_group() {
    u.tok0 = group_ * per_;
    u.ntok = min(per_, u.g.q_len - u.tok0);
    u.tiles = group_tiles(u.g.q_len, u.g.k_len, group_);
  }

  const AttnParams& p_;
  int per_, at_, end_, u0_, group_;
};

// The softmax1 kernels exponentiate a row against a reference m that follows its
// maximum lazily, and round P to the inputs' type.  In float16 the reference is
// kept kHeadroom16 octaves below the maximum that set it: P of that key is 2^8,
// and P down to 2^-22 of it is a normal number.  Rows that attend to almost
// nothing (all scores far below the implicit zero logit) so have references
// below zero.  kLowestRef keeps 2^-m finite: such a row's output is zero in
// float16 as well.  top: the maximum, -inf when there is none (m: 0).
constexpr float kHeadroom16 = 8.f, kLowestRef = -100.f;
__device__ __forceinline__ float reference16(float top) {
  return top > kNegInf ? fmaxf(top - kHeadroom16, kLowestRef) : 0.f;
}

// Integers in the order of the floats; its own inverse on the bits.
__device__ __forceinline__ int ordered_int(float x) {
  const int i = __float_as_int(x);
  return i ^ ((i >> 31) & 0x7fffffff);
}

// Statistics (reference max(m, 0), denominator with the implicit zero logit) of
// a row with reference m and sum l, and the factor of its unscaled output.
struct RowEnd {
  float m, l, inv;
};
template <bool BF16>
__device__ __forceinline__ RowEnd end_of_row(float m, float l) {
  if (BF16) {  // (m >= 0)
    l += exp2f(-m);
    return RowEnd{m, l, 1.f / l};
  }
  const float top = fmaxf(m, 0.f), scale = exp2f(m - top);
  l = l * scale + exp2f(-top);
  return RowEnd{top, l, scale / l};
}

// Joins the pieces of split units: one block per (token, KV head) and its G rows.
// Tokens that no sequence owns get theirs here.
template <int HD, typename T>
__global__ void __launch_bounds__(128) combine_pieces_kernel(const AttnParams p, const PieceWs ws, int group) {
  tc::allow_dependents();
  tc::wait_for_predecessor();  // (set up while the pieces are still being computed)
  const int tok = blockIdx.x / p.hkv, kvh = blockIdx.x % p.hkv;
  const int4 f = ws.info[blockIdx.x];
  if (UnownedRows(p).holds(tok)) {
    store_empty_rows<T, uint2>(p, tok, kvh * group, group);
    return;
  }
  // (under offsets that decrease a token may have no info: kept inside the workspace)
  const int quota = max(f.w, 1), first = min(max(f.x / quota, 0), ws.ctas - 1);
  const int last = min(max((f.x + f.y - 1) / quota, first), ws.ctas - 1);
  if (last == first) return;
  const int head = 2 * first + (f.x == first * quota ? 0 : 1);  // slot of the unit's first piece; the others lead their CTA
  constexpr int LPR = HD / 4;  // lanes of a row: they also share the row's (m, l) loads
  const int parts = last - first + 1, lane = threadIdx.x % LPR, d = lane * 4;
  const unsigned mask = LPR == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
  for (int g = threadIdx.x / LPR; g < group; g += 128 / LPR) {
    const int row = min(max(f.z, 0), ws.rows - group) + g;
    auto at = [&](int j) { return (int64_t)(j == 0 ? head : 2 * (first + j)) * ws.rows + row; };
    float m = 0.f, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = lane; j < parts; j += LPR) m = fmaxf(m, ws.ml[at(j)].x);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(mask, m, o, LPR));
    for (int j0 = 0; j0 < parts; j0 += LPR) {
      const float2 ml = j0 + lane < parts ? ws.ml[at(j0 + lane)] : make_float2(kNegInf, 0.f);
      const float sj = exp2f(ml.x - m);
      l += ml.y * sj;
      const int n = min(LPR, parts - j0);
#pragma unroll 8
      for (int j = 0; j < n; ++j) {
        const float4 x = *reinterpret_cast<const float4*>(ws.o + at(j0 + j) * HD + d);
        const float s = __shfl_sync(mask, sj, j, LPR);
        acc.x = fmaf(s, x.x, acc.x);
        acc.y = fmaf(s, x.y, acc.y);
        acc.z = fmaf(s, x.z, acc.z);
        acc.w = fmaf(s, x.w, acc.w);
      }
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) l += __shfl_xor_sync(mask, l, o, LPR);
    l += exp2f(-m);  // the implicit zero logit
    const float inv = 1.f / l;
    const int h = kvh * group + g;
    if (d == 0) {
      p.stats[(int64_t)h * p.rows_total + tok] = m;
      p.stats[(int64_t)(p.hq + h) * p.rows_total + tok] = l;
    }
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    uint2 y;
    y.x = tc::pack2<BF16>(acc.x * inv, acc.y * inv);
    y.y = tc::pack2<BF16>(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + (int64_t)tok * p.o_st + (int64_t)h * p.o_sh + d) = y;
  }
}

struct PieceLayout {
  int64_t o, ml, info, total;
};
inline PieceLayout piece_layout(const AttnParams& p, int ctas, int rows) {
  auto up = [](int64_t x) { return (x + 255) & ~int64_t(255); };
  PieceLayout w;
  w.o = 0;
  w.ml = up((int64_t)2 * ctas * rows * p.d * 4);
  w.info = w.ml + up((int64_t)2 * ctas * rows * 8);
  w.total = w.info + up((int64_t)p.rows_total * p.hkv * 16);
  return w;
}
inline PieceWs piece_ws(const AttnParams& p, int ctas, int rows, void* workspace) {
  const PieceLayout w = piece_layout(p, ctas, rows);
  uint8_t* base = static_cast<uint8_t*>(workspace);
  return PieceWs{reinterpret_cast<float*>(base + w.o), reinterpret_cast<float2*>(base + w.ml),
                 reinterpret_cast<int4*>(base + w.info), rows, ctas};
}

}  // namespace hfan
