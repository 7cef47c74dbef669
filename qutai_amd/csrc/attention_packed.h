// Attention of packed bf16 sequences with heads of up to 128 channels (multiples
// of 8) on the matrix cores, forward and backward.
//
// A wave takes 32 queries of one head (forward, dQ) or 32 keys of one kv head (dK,
// dV); the other side streams through LDS in blocks of 64 rows, copied with
// buffer_load ... lds into a ring of two stages while the block before is worked
// on.  Scores are computed transposed (S^T = K Q^T with v_mfma_f32_32x32x16_bf16),
// so that a lane holds one query, the softmax's maximum and sum are its own (and
// its partner lane's), and the probabilities are the next product's operand as they
// stand.
//
// The waves of a workgroup share the stream.  They take the query heads of one kv
// head first and consecutive blocks of 32 queries after that: with four heads to a
// kv head a query tile is 32 rows of four heads instead of 128 of one.  Short
// documents then fill tiles (70 documents of 10 to 1024 tokens: 547 tiles of 32 hold
// 17504 rows for 16384 tokens, 168 of 128 21504), and all waves of a causal tile end
// their work together.
//
// What bounds them, 16384 tokens of those documents, 16 heads over 4 of 64, causal:
// forward 49 us (350 TFLOP/s, 2.4 TB/s), dQ 60 (430, 3.1), dK and dV 75 (450): the
// softmax's vector instructions (three and an exponential for each score) beside the
// matrix ones, and each wave's own beginning and end, 40% of the forward's vector
// instructions at 160 visible keys to a query.  16000 tokens of three documents, 32
// heads over 8 of 128: 712 us (990 TFLOP/s), 960 (1100) and 1580 (890; V of the
// wave's keys read from LDS): the matrix cores, where a product of 8192^3 reaches 1160.
//
// Roundings to fewer bits: the probabilities and dS go into the second products as
// bf16 (2^-8 of each, of random sign, as their other operand has; the normaliser
// sums them in fp32; in two parts for sequences of up to FINE tokens), everything else
// stays fp32 until a result is stored.  out's
// own rounding is returned as a second bf16 (`rest`), from which the backward sums
// delta = dO . (out + rest): documents of a few tokens would otherwise see that
// rounding as an error of all their dS (1.2 times the error of dQ and dK).
//
// A wave whose sums hold an infinity or NaN (its operands did, masked or not)
// computes its rows again one at a time (attention_rows.h), where what is masked is
// not read.
#pragma once
#include "attention_rows.h"
#include "attention_mma.h"

namespace {

// Heads of a kv head that share a workgroup of NW waves: the largest power of two.
constexpr int packed_heads(int64_t heads, int64_t kv_heads, int waves) {
  int n = 1;
  while (2 * n <= waves && heads / kv_heads % (2 * n) == 0) n *= 2;
  return n;
}

typedef __attribute__((address_space(3))) const char* lds_bytes;
__device__ __forceinline__ lds_bytes lds_at(const void* x) {
  return (lds_bytes)(lds_ptr_t)const_cast<void*>(x);
}

// DP: channels in steps of 32 that hold a head's.  Heads of 65 to 96 have kernels of their
// own rather than those of 128: dK and dV of 8000 tokens, 16 heads over 4 of 96, 132 us
// (178), dQ 68 (75), forward 61 (65); heads of up to 32 rather than those of 64: 16384
// tokens, 16 over 4 of 32, 53 (72), 36 (48), 30 (39).
template <int DP>
struct PackedTile {
  static constexpr int S = DP / 16, DB = DP / 32;  // MFMA k-steps over d, 32-wide d blocks
  static constexpr int PC = DP > 64 ? 16 : DP / 8;  // 16-byte chunks of a row in LDS, a power of two
  static constexpr int LP = PC * 8, ROW = LP * 2;  // a row in LDS: elements, bytes

  // Chunk c of row r lies at c ^ swz(r).  16 rows' same chunk (a read of 16 lanes) and 4
  // rows' 64 bytes (a transposed read of 32) fall into different banks, and rows 16
  // apart are swizzled alike, so that a lane's addresses in a tile differ by constants.
  __device__ static __forceinline__ int swz(int r) {
    if constexpr (PC == 4) return r >> 2 & 3;
    else if constexpr (PC == 8) return (r >> 1 & 1) << 2 | (r >> 2 & 1) << 1 | (r >> 3 & 1);
    else return (r & 3) << 2 | (r >> 2 & 3);
  }

  // A lane's byte offsets in a tile: of its 16 bytes of row col (row fragments: the
  // 32 s bytes of k-step s are a xor of the chunk), and of its 8 bytes of the two rows of
  // a transposed read (the 64 db bytes of a d block too).
  struct Lane {
    uint32_t row, c0, c1;
    __device__ __forceinline__ void plan(int lane) {
      const int half = lane >> 5, col = lane & 31, g = lane >> 4, i = lane & 15;
      const int r0 = 4 * (g >> 1) + (i >> 2), r1 = r0 + 8, c = 2 * (g & 1) + ((i & 3) >> 1), b = 8 * (i & 1);
      row = col * ROW + (half ^ swz(col)) * 16;
      c0 = r0 * ROW + (c ^ swz(r0)) * 16 + b;
      c1 = r1 * ROW + (c ^ swz(r1)) * 16 + b;
    }
    // The same in the other stage of the ring, BYTES (a power of two) away.
    template <int BYTES>
    __device__ __forceinline__ void flip() {
      row ^= BYTES, c0 ^= BYTES, c1 ^= BYTES;
    }
  };
  // Row fragment: row rb + col, d = 16 s + 8 half + [0, 8), of the tile at x.
  __device__ static __forceinline__ bf16x8 rows(lds_bytes x, const Lane& l, int rb, int s) {
    typedef __attribute__((address_space(3))) const bf16x8* ptr;
    return *(ptr)(x + (l.row ^ (32 * s)) + rb * ROW);
  }
  // Transposed fragment: rows = d columns 32 db + [0, 32), k = tile rows
  // rb + {4 half + [0, 4), 8 + ...}, the order of an MFMA result's elements.
  __device__ static __forceinline__ bf16x8 columns(lds_bytes x, const Lane& l, int db, int rb) {
    typedef __attribute__((address_space(3))) i16x4* ptr;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(x + (l.c0 ^ (64 * db)) + rb * ROW));
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(x + (l.c1 ^ (64 * db)) + rb * ROW));
    const i16x8 w = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8, w);
  }

  // Copies of a block of ROWS rows by NW waves: chunk (j * NW + wave) * 64 + lane of
  // the block, at c ^ swz(r) of row r.
  template <int ROWS, int NW>
  struct Copy {
    static constexpr int N = ROWS * PC / 64 / NW;
    static_assert(N * NW * 64 == ROWS * PC, "whole copies");
    uint32_t off[N];
    int row[N];
    __device__ __forceinline__ void plan(int64_t pitch, int D, int wave, int lane) {
#pragma unroll
      for (int j = 0; j < N; j++) {
        const int at = (j * NW + wave) * 64 + lane, r = at / PC, c = (at % PC) ^ swz(r);
        row[j] = r;
        off[j] = (uint32_t)((r * pitch + 8 * c) * 2) | (8 * c < D ? 0u : ATTN_OOB);
      }
    }
    // rows at or beyond `left` and channels at or beyond D arrive as zeros
    __device__ __forceinline__ void issue(bf16_t* to, const bf16_t* from, int64_t pitch, int left, int wave) const {
      const u32x4 r = lds_rsrc(from, ROWS * pitch * 2);
#pragma unroll
      for (int j = 0; j < N; j++)
        lds_load16(r, reinterpret_cast<char*>(to) + (j * NW + wave) * 1024, off[j] | (row[j] < left ? 0u : ATTN_OOB));
    }
  };

  // The wave's own 32 rows as operands: lane = row col, d = 16 s + 8 half + [0, 8).
  __device__ static __forceinline__ void own(const void* base, int64_t first, int64_t pitch, int left, int D, int col,
                                             int half, bf16x8 (&f)[S]) {
    const auto r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<bf16_t*>(uniform_ptr((const bf16_t*)base + first)), 0, (uint32_t)(32 * pitch * 2), 0x00020000);
#pragma unroll
    for (int s = 0; s < S; s++) {
      const int d = 16 * s + 8 * half;
      const uint32_t off = (uint32_t)((col * pitch + d) * 2) | (col < left && d < D ? 0u : ATTN_OOB);
      f[s] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
    }
  }
};

__device__ __forceinline__ bf16x8 rounded(const float* v) {
  const u32x4 w = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
  return __builtin_bit_cast(bf16x8, w);
}

// What `rounded` left of the same values, as bf16 again.
__device__ __forceinline__ bf16x8 left_of(const float* v, const bf16x8& kept) {
  const u32x4 w = __builtin_bit_cast(u32x4, kept);
  float r[8];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    r[2 * i] = v[2 * i] - __uint_as_float(w[i] << 16);
    r[2 * i + 1] = v[2 * i + 1] - __uint_as_float(w[i] & 0xffff0000u);
  }
  return rounded(r);
}

// Sequences that are not longer take probabilities and dS into their products in two bf16
// parts, whatever lies beside them: the few roundings of short sums do not average out (87
// tokens of sequences of up to 6: dQ 1.5 times as far off as in fp32), and the products are
// not what bounds them.  In the query passes every masked block carries two parts (all blocks
// of such sequences take the masked form; those on the diagonal or at the end of longer ones
// gain by it for 0 to 4% of the time, most for the forward of one document of 2000 tokens, 16
// heads over 4 of 128, 57 us and 55), in the key pass a loop of its own, which is all that a
// batch of only such sequences needs (ONLY).  Forward, dQ, dK and dV in two parts and in one,
// us: 16384 tokens of up to 64, 16 heads over 4 of 64, 40 and 38, 44 and 42, 60 and 60; 16000,
// 32 over 8 of 128, 143 and 141, 220 and 215, 173 and 203.
constexpr int FINE = 64;

// x += the 32 tile rows from `row` on, transposed, times the lane's weights of them, rounded
// to bf16, and with PARTS what that rounding leaves.  Two parts of wide heads: one half of
// the weights after the other, whose registers are free sooner (16000 tokens of up to 64, 32
// heads over 8 of 128, dK and dV: 173 us, 208 with both halves of each d block together).
template <int DP, bool PARTS>
__device__ __forceinline__ void add_columns(lds_bytes tile, const typename PackedTile<DP>::Lane& at, int row,
                                            const float (&w)[16], f32x16 (&x)[DP / 32]) {
  const bf16x8 kept[2] = {rounded(w), rounded(w + 8)};
  bf16x8 left[2];
  auto add = [&](int db, int st) {
    const bf16x8 v = PackedTile<DP>::columns(tile, at, db, row + 16 * st);
    if constexpr (PARTS) x[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, left[st], x[db], 0, 0, 0);
    x[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, kept[st], x[db], 0, 0, 0);
  };
  if constexpr (PARTS && DP > 64) {
#pragma unroll
    for (int st = 0; st < 2; st++) {
      left[st] = left_of(w + 8 * st, kept[st]);
#pragma unroll
      for (int db = 0; db < DP / 32; db++) add(db, st);
    }
  } else {
    if constexpr (PARTS) left[0] = left_of(w, kept[0]), left[1] = left_of(w + 8, kept[1]);
#pragma unroll
    for (int db = 0; db < DP / 32; db++) add(db, 0), add(db, 1);
  }
}

// All waves have a block in LDS and are done with the one before, whose stage is copied into
// next: a wave's reads of it, and what it wrote, are waited for here, wherever the compiler
// puts their uses.
__device__ __forceinline__ void stage_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The tile, heads and rows of a wave of a query tile.
struct PackedPlace {
  int h, kvh, first, q0;  // first row of the tile, of the wave
};
template <int NW>
__device__ __forceinline__ PackedPlace enter_queries(AttnPackedArgs& p, int wave) {
  const int pack = p.pack, subs = (int)p.heads / pack;
  const int tile = uniform32((int)blockIdx.x / subs), h0 = uniform32((int)blockIdx.x % subs) * pack;
  PackedPlace at;
  at.first = enter_sequence<bf16_t>(p, tile);
  at.h = uniform32(h0 + wave % pack);
  at.kvh = uniform32(h0 / (int)(p.heads / p.kv_heads));
  at.q0 = uniform32(at.first + wave / pack * 32);
  return at;
}

// HALVES times 32 keys from row 32 mb of the block on, for the wave's queries: all
// scores first, so that the later halves' products overlap the first half's
// exponentials.  lim (MASK): the keys of the block that the lane's query sees, less 4 half.
template <int DP, int HALVES, bool MASK>
__device__ __forceinline__ void packed_attend(lds_bytes sk, lds_bytes sv, const typename PackedTile<DP>::Lane& at,
                                              const bf16x8 (&qf)[DP / 16], f32x16 (&o)[DP / 32], float& m, float& l,
                                              int lim, float c, int mb) {
  typedef PackedTile<DP> Tile;
  f32x16 sc[HALVES];
  float peak = -INFINITY;
#pragma unroll
  for (int n = 0; n < HALVES; n++) {
    sc[n] = f32x16{};
#pragma unroll
    for (int s = 0; s < Tile::S; s++)
      sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(Tile::rows(sk, at, 32 * (mb + n), s), qf[s], sc[n], 0, 0, 0);
  }
#pragma unroll
  for (int n = 0; n < HALVES; n++) {
    if constexpr (MASK) {
#pragma unroll
      for (int e = 0; e < 16; e++)
        if (32 * (mb + n) + 8 * (e >> 2) + (e & 3) >= lim) sc[n][e] = -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 16; e++) peak = fmaxf(peak, sc[n][e]);
  }
  // the reference point m moves only for a maximum more than 2^8 above it
  const float cand = pair_max(peak) * c;
  const bool grow = cand > m + 8.f;
  if (__builtin_amdgcn_ballot_w64(grow)) {
    if (grow) {
      const float alpha = __builtin_amdgcn_exp2f(m - cand);
      m = cand;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < Tile::DB; db++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[db][e] *= alpha;
    }
  }
  const float ref = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int n = 0; n < HALVES; n++) {
    float pv[16];
#pragma unroll
    for (int e = 0; e < 16; e++) {
      pv[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][e], c, -ref));
      sum += pv[e];
    }
    add_columns<DP, MASK>(sv, at, 32 * (mb + n), pv, o);
  }
  l += sum;
}

// Four consecutive channels of a result row, and of what its rounding left.
__device__ __forceinline__ void put_rest(void* base, int64_t at, const f32x4& v, const u32x2& stored) {
  const f32x4 kept = {__uint_as_float(stored[0] << 16), __uint_as_float(stored[0] & 0xffff0000u),
                      __uint_as_float(stored[1] << 16), __uint_as_float(stored[1] & 0xffff0000u)};
  const f32x4 left = v - kept;
  global_store((bf16_t*)base + at, u32x2{pack_bf16x2(left[0], left[1]), pack_bf16x2(left[2], left[3])});
}

template <int DP, int NW, int KB>
__global__ void __launch_bounds__(NW * 64, DP <= 64 ? 4 : 3) packed_fwd(AttnPackedArgs p) {
  typedef PackedTile<DP> Tile;
  __shared__ __attribute__((aligned(16))) bf16_t lds[2][2][KB * Tile::LP];  // [stage][K, V]
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform32(tid >> 6), half = lane >> 5, col = lane & 31;
  const PackedPlace at = enter_queries<NW>(p, wave);
  const int T = (int)p.time, D = (int)p.dim, q0 = at.q0, t = q0 + col, tile_rows = NW / p.pack * 32;
  const bf16_t* K = uniform_ptr((const bf16_t*)p.k + at.kvh * p.kh);
  const bf16_t* V = uniform_ptr((const bf16_t*)p.v + at.kvh * p.kh);

  bf16x8 qf[Tile::S];
  Tile::own(p.q, at.h * p.qh + (int64_t)q0 * p.qt, p.qt, T - q0, D, col, half, qf);
  typename Tile::template Copy<KB, NW> ck, cv;
  ck.plan(p.kt, D, wave, lane);
  cv.plan(p.vt, D, wave, lane);
  auto issue = [&](int kbk) {
    const int64_t kv0 = (int64_t)kbk * KB;
    ck.issue(&lds[kbk & 1][0][0], K + kv0 * p.kt, p.kt, T - kbk * KB, wave);
    cv.issue(&lds[kbk & 1][1][0], V + kv0 * p.vt, p.vt, T - kbk * KB, wave);
  };

  f32x16 o[Tile::DB];
#pragma unroll
  for (int db = 0; db < Tile::DB; db++) o[db] = f32x16{};
  float m = -INFINITY, l = 0.f;
  const float c = p.scale_log2;
  // blocks of which the wave's queries see every key, halves of blocks of which they
  // see some, blocks of which they see none (the copies' and barriers' order is kept)
  const int nkb = ((p.causal ? min(at.first + tile_rows, T) : T) + KB - 1) / KB;
  const int seen = q0 >= T ? 0 : p.causal ? min(q0 + 32, T) : T;
  const int n_full = T <= FINE ? 0 : min(seen, p.causal ? q0 + 1 : T) / KB;
  auto advance = [&](int kbk) {  // wait for a block, start the next one's copies
    wait_vmcnt<0>();
    stage_barrier();
    if (kbk + 1 < nkb) issue(kbk + 1);
  };
  if (nkb > 0) issue(0);
  constexpr int STAGE = 2 * KB * Tile::ROW;
  typename Tile::Lane in;  // in the stage of block kbk
  in.plan(lane);
  const lds_bytes sk = lds_at(&lds[0][0][0]), sv = lds_at(&lds[0][1][0]);
  int kbk = 0;
  for (; kbk < n_full; kbk++) {
    advance(kbk);
    packed_attend<DP, KB / 32, false>(sk, sv, in, qf, o, m, l, 0, c, 0);
    in.template flip<STAGE>();
  }
  for (; kbk * KB < seen; kbk++) {
    advance(kbk);
    const int kv0 = kbk * KB, lim = min(T - kv0, p.causal ? t - kv0 + 1 : KB) - 4 * half;
#pragma unroll 1
    for (int mb = 0; mb < KB / 32 && kv0 + 32 * mb < seen; mb++)
      packed_attend<DP, 1, true>(sk, sv, in, qf, o, m, l, lim, c, mb);
    in.template flip<STAGE>();
  }
  for (; kbk < nkb; kbk++) advance(kbk);

  const float total = pair_sum(l);
  const float bad = not_finite(o) + total * 0.f + m * 0.f;
  if (__builtin_amdgcn_ballot_w64(t < T && !(bad == 0.f))) {
    for (int i = 0; i < 32 && q0 + i < T; i++) {
      fwd_row<bf16_t>(p, 0, at.h, q0 + i, lane);
      if (p.rest)
        for (int d = lane; d < D; d += 64) ((bf16_t*)p.rest)[at.h * p.qh + (int64_t)(q0 + i) * p.ot + d] = 0;
    }
    return;
  }
  if (t < T) {
    const float inv = 1.f / total;
    const int64_t to = at.h * p.qh + (int64_t)t * p.ot;
#pragma unroll
    for (int db = 0; db < Tile::DB; db++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int d = 32 * db + 8 * g + 4 * half;
        if (d >= D) continue;
        const f32x4 v = f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]} * inv;
        const u32x2 w = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        global_store((bf16_t*)p.dq + to + d, w);
        if (p.rest) put_rest(p.rest, to + d, v, w);
      }
    if (half == 0) p.lse[at.h + t * p.lt] = (m + __log2f(total)) * 0.6931471805599453f;
  }
}

// dQ of the wave's queries, and delta; K and V stream.
template <int DP, bool MASK>
__device__ __forceinline__ void packed_dq_step(lds_bytes sk, lds_bytes sv, const typename PackedTile<DP>::Lane& at,
                                               const bf16x8 (&qf)[DP / 16], const bf16x8 (&gf)[DP / 16], float lse2,
                                               float dl, f32x16 (&dqt)[DP / 32], int lim, float c, int mb) {
  typedef PackedTile<DP> Tile;
  f32x16 sc = {}, dp = {};
#pragma unroll
  for (int s = 0; s < Tile::S; s++) {
    sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(Tile::rows(sk, at, 32 * mb, s), qf[s], sc, 0, 0, 0);
    dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(Tile::rows(sv, at, 32 * mb, s), gf[s], dp, 0, 0, 0);
  }
  float ds[16];
#pragma unroll
  for (int e = 0; e < 16; e++) {
    float x = sc[e];
    if constexpr (MASK)
      if (32 * mb + 8 * (e >> 2) + (e & 3) >= lim) x = -INFINITY;
    ds[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c, -lse2)) * (dp[e] - dl);
  }
  if constexpr (MASK) __builtin_amdgcn_sched_barrier(0);  // six registers less to spill: 44 us, not 48, on 16384 tokens of up to 64
  add_columns<DP, MASK>(sk, at, 32 * mb, ds, dqt);
}

template <int DP, int NW>
__global__ void __launch_bounds__(NW * 64, DP <= 64 ? 4 : 2) packed_bwd_dq(AttnPackedArgs p) {
  typedef PackedTile<DP> Tile;
  constexpr int KB = 64;
  __shared__ __attribute__((aligned(16))) bf16_t lds[2][2][KB * Tile::LP];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform32(tid >> 6), half = lane >> 5, col = lane & 31;
  const PackedPlace at = enter_queries<NW>(p, wave);
  const int T = (int)p.time, D = (int)p.dim, q0 = at.q0, t = q0 + col, tile_rows = NW / p.pack * 32;
  const bf16_t* K = uniform_ptr((const bf16_t*)p.k + at.kvh * p.kh);
  const bf16_t* V = uniform_ptr((const bf16_t*)p.v + at.kvh * p.kh);
  const int64_t head = at.h * p.qh;

  bf16x8 qf[Tile::S], gf[Tile::S];
  float dl = 0.f, lse2 = 0.f;
  {
    Tile::own(p.g, head + (int64_t)q0 * p.ot, p.ot, T - q0, D, col, half, gf);
    // delta: the diagonal of O dO^T, summed as dP is, so that a query that sees one
    // key leaves what O and V leave, and of the rest
    f32x16 og = {};
    Tile::own(p.o, head + (int64_t)q0 * p.ot, p.ot, T - q0, D, col, half, qf);
#pragma unroll
    for (int s = 0; s < Tile::S; s++) og = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf[s], gf[s], og, 0, 0, 0);
    if (p.rest) {
      Tile::own(p.rest, head + (int64_t)q0 * p.ot, p.ot, T - q0, D, col, half, qf);
#pragma unroll
      for (int s = 0; s < Tile::S; s++) og = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf[s], gf[s], og, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 16; e++)
      if (8 * (e >> 2) + 4 * half + (e & 3) == col) dl = og[e];
    dl = pair_sum(dl);
    const int64_t li = at.h + (int64_t)t * p.lt;
    if (t < T) lse2 = p.lse[li] * LOG2E;
    if (t < T && half == 0) p.delta[li] = dl;
    Tile::own(p.q, head + (int64_t)q0 * p.qt, p.qt, T - q0, D, col, half, qf);
  }
  typename Tile::template Copy<KB, NW> ck, cv;
  ck.plan(p.kt, D, wave, lane);
  cv.plan(p.vt, D, wave, lane);
  auto issue = [&](int kbk) {
    const int64_t kv0 = (int64_t)kbk * KB;
    ck.issue(&lds[kbk & 1][0][0], K + kv0 * p.kt, p.kt, T - kbk * KB, wave);
    cv.issue(&lds[kbk & 1][1][0], V + kv0 * p.vt, p.vt, T - kbk * KB, wave);
  };
  f32x16 dqt[Tile::DB];
#pragma unroll
  for (int db = 0; db < Tile::DB; db++) dqt[db] = f32x16{};
  const float c = p.scale_log2;
  const int nkb = ((p.causal ? min(at.first + tile_rows, T) : T) + KB - 1) / KB;
  const int seen = q0 >= T ? 0 : p.causal ? min(q0 + 32, T) : T;
  const int n_full = T <= FINE ? 0 : min(seen, p.causal ? q0 + 1 : T) / KB;
  auto advance = [&](int kbk) {
    wait_vmcnt<0>();
    stage_barrier();
    if (kbk + 1 < nkb) issue(kbk + 1);
  };
  if (nkb > 0) issue(0);
  constexpr int STAGE = 2 * KB * Tile::ROW;
  typename Tile::Lane in;  // in the stage of block kbk
  in.plan(lane);
  const lds_bytes sk = lds_at(&lds[0][0][0]), sv = lds_at(&lds[0][1][0]);
  int kbk = 0;
  for (; kbk < n_full; kbk++) {
    advance(kbk);
#pragma unroll 1
    for (int mb = 0; mb < 2; mb++) packed_dq_step<DP, false>(sk, sv, in, qf, gf, lse2, dl, dqt, 0, c, mb);
    in.template flip<STAGE>();
  }
  for (; kbk * KB < seen; kbk++) {
    advance(kbk);
    const int kv0 = kbk * KB, lim = min(T - kv0, p.causal ? t - kv0 + 1 : KB) - 4 * half;
#pragma unroll 1
    for (int mb = 0; mb < 2 && kv0 + 32 * mb < seen; mb++)
      packed_dq_step<DP, true>(sk, sv, in, qf, gf, lse2, dl, dqt, lim, c, mb);
    in.template flip<STAGE>();
  }
  for (; kbk < nkb; kbk++) advance(kbk);

  if (__builtin_amdgcn_ballot_w64(t < T && !(not_finite(dqt) + dl * 0.f == 0.f))) {
    for (int i = 0; i < 32 && q0 + i < T; i++) bwd_q_row<bf16_t>(p, 0, at.h, q0 + i, lane);
    return;
  }
  if (t < T) {
    const int64_t to = head + (int64_t)t * p.dqt;
#pragma unroll
    for (int db = 0; db < Tile::DB; db++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int d = 32 * db + 8 * g + 4 * half;
        if (d < D)
          put4<false>(p.dq, to + d, f32x4{dqt[db][4 * g], dqt[db][4 * g + 1], dqt[db][4 * g + 2], dqt[db][4 * g + 3]} * p.scale);
      }
  }
}

// A key tile: waves of 32 keys; QB: rows of a streamed block.  Two sums of 128
// channels and K and V of the wave's keys do not fit 256 registers beside the scores
// (97 of them spilled): there V stays in LDS, for 8 reads more beside 32 products.
// Blocks of 32 rows leave room for two workgroups on a CU.
// Heads of up to 32 leave registers for three waves of a SIMD (16384 tokens, 53 us; for
// four, with 20 spilled, 62).
template <int DP>
struct PackedKeys {
  static constexpr int QB = DP > 64 ? 32 : 64;
  static constexpr bool V_IN_LDS = DP > 96;
  static constexpr int VF = V_IN_LDS ? 1 : DP / 16;
};

// dK and dV of the wave's 32 keys: 32 queries from row 32 mb of the streamed block
// on.  Element e of a score block: query 32 mb + 8 (e / 4) + 4 half + e % 4, key col.
// One product after the other, so that dK's and dV's sums, the wave's K and V and
// one block of scores and dP are all that lives.
template <int DP, bool MASK, bool PARTS>
__device__ __forceinline__ void packed_dkv_step(lds_bytes sq, lds_bytes sg, const typename PackedTile<DP>::Lane& at,
                                                const float* slse, const float* sdl, const bf16x8 (&kf)[DP / 16],
                                                const bf16x8 (&vf)[PackedKeys<DP>::VF], lds_bytes sv,
                                                const typename PackedTile<DP>::Lane& own, f32x16 (&dkt)[DP / 32],
                                                f32x16 (&dvt)[DP / 32], int end, int before, float c, int half, int mb) {
  typedef PackedTile<DP> Tile;
  f32x16 sc = {};
#pragma unroll
  for (int s = 0; s < Tile::S; s++)
    sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(Tile::rows(sq, at, 32 * mb, s), kf[s], sc, 0, 0, 0);
  if constexpr (DP > 64) __builtin_amdgcn_sched_barrier(0);
  float pr[16];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const f32x4 l4 = *reinterpret_cast<const f32x4*>(slse + 32 * mb + 8 * j + 4 * half);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float x = sc[4 * j + i];
      if constexpr (MASK) {
        const int q = 32 * mb + 8 * j + 4 * half + i;
        if (q >= end || q < before) x = -INFINITY;  // before: of a causal key
      }
      pr[4 * j + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c, l4[i]));  // slse holds -lse log2(e)
    }
  }
  add_columns<DP, PARTS>(sg, at, 32 * mb, pr, dvt);
  if constexpr (DP > 64) __builtin_amdgcn_sched_barrier(0);
  f32x16 dp = {};
#pragma unroll
  for (int s = 0; s < Tile::S; s++)
    dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(Tile::rows(sg, at, 32 * mb, s),
                                                 PackedKeys<DP>::V_IN_LDS ? Tile::rows(sv, own, 0, s)
                                                                          : vf[PackedKeys<DP>::V_IN_LDS ? 0 : s],
                                                 dp, 0, 0, 0);
  if constexpr (DP > 64) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const f32x4 d4 = *reinterpret_cast<const f32x4*>(sdl + 32 * mb + 8 * j + 4 * half);
#pragma unroll
    for (int i = 0; i < 4; i++) pr[4 * j + i] *= dp[4 * j + i] - d4[i];
  }
  add_columns<DP, PARTS>(sq, at, 32 * mb, pr, dkt);
}

// SPLIT sets of KW waves take the query heads of a group in turns, each with a stream
// of its own, and add up their sums at the end in the order of the sets.  ONLY: no sequence
// has more than FINE tokens (us with the loops of longer ones in the kernel too: 16384 tokens
// of up to 64, 16 heads over 4 of 64, 65 instead of 60; 8000, 16 over 4 of 96, 43 and 29).
template <int DP, int KW, int SPLIT, bool ONLY = false>
__global__ void __launch_bounds__(KW * SPLIT * 64, DP == 32 ? 3 : 2) packed_bwd_dkv(AttnPackedArgs p) {
  typedef PackedTile<DP> Tile;
  constexpr int QB = PackedKeys<DP>::QB;
  constexpr bool V_IN_LDS = PackedKeys<DP>::V_IN_LDS;
  __shared__ __attribute__((aligned(16))) bf16_t lds[2][SPLIT][2][QB * Tile::LP];  // [stage][set][Q, dO]
  __shared__ __attribute__((aligned(16))) float stats[2][SPLIT][2][QB];      // [stage][set][-lse log2(e), delta]
  __shared__ __attribute__((aligned(16))) bf16_t own_v[V_IN_LDS ? KW * 32 * Tile::LP : 8];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int set = uniform32(tid >> 6) / KW, wave = uniform32(tid >> 6) % KW;
  const int group = (int)(p.heads / p.kv_heads);
  int b, kvh, blk, gsel;
  place_keys<bf16_t, 1>(p, 1, b, kvh, blk, gsel);
  const int T = (int)p.time, D = (int)p.dim, k0 = blk, kw = uniform32(k0 + wave * 32), key = kw + col;

  bf16x8 kf[Tile::S], vf[PackedKeys<DP>::VF];
  Tile::own(p.k, kvh * p.kh + (int64_t)kw * p.kt, p.kt, T - kw, D, col, half, kf);
  if constexpr (V_IN_LDS) {  // there before the first block is, whose wait and barrier cover it
    if (set == 0) {
      typename Tile::template Copy<KW * 32, KW> cv;
      cv.plan(p.vt, D, wave, lane);
      cv.issue(own_v, uniform_ptr((const bf16_t*)p.v + kvh * p.kh + (int64_t)k0 * p.vt), p.vt, T - k0, wave);
    }
  } else {
    Tile::own(p.v, kvh * p.kh + (int64_t)kw * p.vt, p.vt, T - kw, D, col, half, vf);
  }
  f32x16 dkt[Tile::DB], dvt[Tile::DB];
#pragma unroll
  for (int db = 0; db < Tile::DB; db++) dkt[db] = dvt[db] = f32x16{};

  // every set makes the same iterations, whose barriers all waves share: heads
  // kvh group + set + SPLIT g (SPLIT divides the group)
  const int qs0 = p.causal ? k0 : 0, nq = (T - qs0 + QB - 1) / QB, iterations = nq * (group / SPLIT);
  typename Tile::template Copy<QB, KW> cq, cg;
  cq.plan(p.qt, D, wave, lane);
  cg.plan(p.ot, D, wave, lane);
  float next = 0.f;  // a set's waves 0 and 1: the lane's row of the block in flight, lse and delta
  auto issue = [&](int it, int h, int qs) {
    bf16_t* to = &lds[it & 1][set][0][0];
    cq.issue(to, uniform_ptr((const bf16_t*)p.q + h * p.qh + (int64_t)qs * p.qt), p.qt, T - qs, wave);
    cg.issue(to + QB * Tile::LP, uniform_ptr((const bf16_t*)p.g + h * p.qh + (int64_t)qs * p.ot), p.ot, T - qs, wave);
    if (wave < 2 && lane < QB) {
      const float* from = wave ? p.delta : p.lse;
      next = qs + lane < T ? from[h + (int64_t)(qs + lane) * p.lt] : 0.f;
    }
  };
  // wait for a block, start the copies of the next one: of the same head, or the
  // first of the set's next
  auto advance = [&](int it, int h, int qi) {
    wait_vmcnt<0>();
    if (wave < 2 && lane < QB) stats[it & 1][set][wave][lane] = wave ? next : -next * LOG2E;
    stage_barrier();
    if (it + 1 < iterations) {
      const bool wrap = qi + 1 == nq;
      issue(it + 1, wrap ? h + SPLIT : h, qs0 + (wrap ? 0 : qi + 1) * QB);
    }
  };
  // steps of 32 queries, per head: before every key of the wave (causal; skipped), all of a
  // short sequence (masked, in two parts), or of a longer one: on the diagonal (masked), with
  // every pair visible, at the sequence's end (masked); behind it (skipped)
  constexpr int HB = QB / 32;
  const int steps = nq * HB, rows = T - qs0;
  auto clamped = [&](int x, int lo) { return x < lo ? lo : x > steps ? steps : x; };
  const bool none = kw >= T;
  const int skipped = none ? steps : p.causal ? clamped((kw - qs0) / 32, 0) : 0;
  const int fine = none || !ONLY && T > FINE ? 0 : clamped((rows + 31) / 32, skipped);
  const int diagonal = none ? steps : T <= FINE ? fine : clamped(p.causal ? skipped + 1 : 0, skipped);
  const int tail = none ? steps : clamped(rows / 32, diagonal);
  const int end = none ? steps : clamped((rows + 31) / 32, tail);
  if (iterations > 0) issue(0, kvh * group + set, qs0);
  constexpr int STAGE = SPLIT * 2 * QB * Tile::ROW;
  typename Tile::Lane in, own;  // in the stage of block `it`, in the wave's rows of V
  in.plan(lane);
  own = in;
  own.row += wave * 32 * Tile::ROW;
  in.template flip<STAGE>();  // as every block's entry does
  const lds_bytes sq = lds_at(&lds[0][set][0][0]), sg = lds_at(&lds[0][set][1][0]), sv = lds_at(own_v);
  int it = -1;
  for (int h = kvh * group + set; h < kvh * group + group; h += SPLIT) {
    auto enter = [&](int st) {
      if (st % HB == 0) {
        advance(++it, h, st / HB);
        in.template flip<STAGE>();
      }
    };
    auto step = [&](int st, auto mask, auto parts) {
      const int qi = st / HB, qs = qs0 + qi * QB;
      packed_dkv_step<DP, decltype(mask)::value, decltype(parts)::value>(
          sq, sg, in, &stats[it & 1][set][0][0], &stats[it & 1][set][1][0], kf, vf, sv, own, dkt, dvt, T - qs,
          p.causal ? key - qs : -1, p.scale_log2, half, st % HB);
    };
    int st = 0;
    for (; st < skipped; st++) enter(st);
    // unlikely: else the registers of this loop are spilled from those below (one document of
    // 2000 tokens, 16 heads over 4 of 128, 171 us instead of 160)
    if (ONLY || __builtin_expect(T <= FINE, 0))
      for (; st < fine; st++) {
        enter(st);
        step(st, std::true_type{}, std::true_type{});
      }
    if constexpr (!ONLY) {
      for (; st < diagonal; st++) {
        enter(st);
        step(st, std::true_type{}, std::false_type{});
      }
      if constexpr (HB > 1) {  // whole blocks, whose two steps overlap
        for (; st < tail && st % HB; st++) {
          enter(st);
          step(st, std::false_type{}, std::false_type{});
        }
        for (; st + HB <= tail; st += HB) {
          enter(st);
          step(st, std::false_type{}, std::false_type{});
          step(st + 1, std::false_type{}, std::false_type{});
        }
      }
      for (; st < tail; st++) {
        enter(st);
        step(st, std::false_type{}, std::false_type{});
      }
      for (; st < end; st++) {
        enter(st);
        step(st, std::true_type{}, std::false_type{});
      }
    }
    for (; st < steps; st++) enter(st);
  }

  if constexpr (SPLIT > 1) {
    // set s hands its sums to set 0 through the stages, 16 channels of dK and dV a turn
    // (4 KiB a wave), in the lanes that hold them
    static_assert(sizeof(lds) >= KW * 64 * 2 * 16 * sizeof(float), "a turn's sums fit the stages");
    f32x16* sums = reinterpret_cast<f32x16*>(&lds[0][0][0][0]) + (wave * 64 + lane) * 2;
#pragma unroll
    for (int from = 1; from < SPLIT; from++)
#pragma unroll
      for (int db = 0; db < Tile::DB; db++) {
        __syncthreads();
        if (set == from) {
          sums[0] = dkt[db];
          sums[1] = dvt[db];
        }
        __syncthreads();
        if (set == 0) {
          dkt[db] += sums[0];
          dvt[db] += sums[1];
        }
      }
    if (set) return;
  }
  const bool bad = key < T && !(not_finite(dkt) + not_finite(dvt) == 0.f);
  if (__builtin_amdgcn_ballot_w64(bad)) {
    for (int i = 0; i < 32 && kw + i < T; i++) bwd_kv_row<bf16_t>(p, 0, kvh, kw + i, lane, 0, group);
    return;
  }
  if (key < T) {
    const int64_t head = kvh * p.kh;
    const int64_t to_k = head + (int64_t)key * p.dkt, to_v = head + (int64_t)key * p.dvt;
#pragma unroll
    for (int db = 0; db < Tile::DB; db++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int d = 32 * db + 8 * g + 4 * half;
        if (d >= D) continue;
        const f32x4 x = {dkt[db][4 * g], dkt[db][4 * g + 1], dkt[db][4 * g + 2], dkt[db][4 * g + 3]};
        const f32x4 y = {dvt[db][4 * g], dvt[db][4 * g + 1], dvt[db][4 * g + 2], dvt[db][4 * g + 3]};
        put4<false>(p.dk, to_k + d, x * p.scale);
        put4<false>(p.dv, to_v + d, y);
      }
  }
}

}  // namespace
