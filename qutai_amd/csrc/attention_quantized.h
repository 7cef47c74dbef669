// Attention of new positions over a quantised key and value cache, on the
// matrix cores (the codes and their layout: cache_codes.h).
//
// The rows of a (sequence, kv head) are its new positions' query heads, row
// t G + j for position t and head j of the G that read the kv head.  A workgroup
// of four waves takes a tile of rows and a range of keys; a wave takes every
// fourth block of 32 keys and keeps a softmax of its own, joined at the end
// of the workgroup; the ranges of a split row are joined by attend_join.
//
// Per block, with v_mfma_f32_16x16x32_bf16 (lane l: column l % 16, row or depth
// group g = l / 16):
//   S^T = K Q^T: the keys are rows; a lane gets keys 4g .. 4g+3 of each 16 for
//   the row (query) of its column;
//   O^T += V^T P^T: the channels are rows; P^T's 8 depths of group g are exactly
//   the 8 scores the lane has (depth j: key 16 (j / 4) + 4g + j % 4), so the
//   probabilities never leave their registers, and V's codes come from 8 rows,
//   w bytes of each, which the conversion to bf16 turns into w operands.
// Codes are integers up to 127: exact in bf16.  The scales stay in fp32: a key's
// multiplies its score, a value's its probability.  Queries and weighted
// probabilities that bf16 does not hold are sums of parts: PARTS of them, two for
// bf16 outputs (16 bits), three for fp32.  Where a tile has few rows (SPREAD > 1)
// the columns hold each row SPREAD times, and the parts of its probabilities go
// into these columns: one product instead of PARTS.  With four rows or fewer of two
// parts (BLOCKS = 2) half of the columns belong to a second block of keys: zeros in
// the operands keep the other block's products out, and what is done with the scores
// and the probabilities is done for both blocks at once (16 sequences of up to 8000
// keys, 4 bits, ranges joined: 42 us with one, 35 with two).
//
// The running maximum of a row is only raised when a score exceeds it by 2^8
// (in powers of two): fp32 holds the sums all the same, and nearly every block
// then runs without an exchange between lanes or a rescaling of the sums.  (So a
// weight is 2^8 at most: sums of up to 2^30 values of 1e27 stay within fp32.)
//
// Bound by HBM with 8 bits and few rows: 32 sequences of up to 16000 keys, 32 heads
// of 128 over 8, 0.67 GB: 128 to 131 us (5.1 TB/s; a wave per query and head 9072), and
// 5 to join.  Bound by vector operations with 4 bits (16 of up to 8000 keys, 92 MB: 34 us,
// and 4 to join)
// and with many rows, where the softmax of a block costs more than its codes (512
// new positions over 3500, 16 heads of 64 over 4: 63 us for 7.4 GFLOP).
#pragma once
#include <type_traits>

#include "cache_codes.h"
#include "qutai_amd.h"

using namespace qa;

namespace {

constexpr int WAVES = 4, BLOCK = 32;  // keys of a block
constexpr float LOWEST = -3.4028234663852886e38f, RISE = 8.f;

struct AttendArgs {
  const void* q;
  const uint8_t* codes[2];
  const bf16_t* scales[2];
  void* out;
  const int64_t* starts;
  const int64_t* counts;
  float* part;  // split rows: [tile][split][rows][pitch] sums, then [tile][split][rows] (maximum, weight)
  float* stats;
  int64_t start, fresh, heads, kv_heads, capacity, units;  // units: sequences x kv heads
  int group, dim, vector, tiles, splits;
  float scale;  // times log2 e
};

struct AttendPlan {
  int tile, spread, rows, pitch;  // row tiles of 16 columns, copies of a row, rows of a workgroup
  int64_t tiles, splits;
};

// Two tiles of such rows do not fit in registers (4 bits, bf16, 256 channels, 512 new positions over 3000: 324 us
// with one, 490 with two; 8 bits 198 and 158).
constexpr bool one_tile(int item, int bits, int pitch) { return item == 4 ? pitch > 128 : bits == 4 && pitch == 256; }

// Blocks of keys beside each other in a tile of four rows or fewer: two, but for wide
// rows of 8 bits, whose operands then leave no room for a second wave (16 sequences
// of up to 7000 keys, 192 channels: 54 us, one 50; 4 bits: 57 and 71).
constexpr int blocks_of(int item, int bits, int pitch) { return item == 2 && (pitch <= 128 || bits == 4) ? 2 : 1; }

template <class T> struct Parts;
template <> struct Parts<bf16_t> { static constexpr int Q = 1, P = 2; };
template <> struct Parts<float> { static constexpr int Q = 3, P = 3; };

// 8 signed bytes as bf16
__device__ __forceinline__ bf16x8 bytes_bf16(uint32_t lo, uint32_t hi) {
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const uint32_t x = e < 2 ? lo : hi;
    w[e] = pack_bf16x2((float)(int8_t)(x >> (16 * (e & 1))), (float)(int8_t)(x >> (16 * (e & 1) + 8)));
  }
  return __builtin_bit_cast(bf16x8, w);
}

__device__ __forceinline__ float scale_at(const uint32_t* w, int i) {
  return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
}

// The channel of operand i's row r (0 .. 15) of the value product, and, for 8
// bits, where a lane's bytes lie: pieces of 16, 8, 4 and 2 bytes per lane.
template <int BITS, int DP>
__device__ __forceinline__ int value_channel(int i, int r) {
  if constexpr (BITS == 4) return 32 * (i >> 1) + 2 * r + (i & 1);
  else if constexpr (DP == 96) return i < 4 ? 4 * r + i : 64 + 2 * r + i - 4;
  else if constexpr (DP == 192) return i < 8 ? 8 * r + i : 128 + 4 * r + i - 8;
  else return DP / 16 * r + i;
}

// Loads take a base that is the same for the wave and a lane's 32-bit offset: no
// 64-bit addresses in vector registers.

// the bytes of a key's value row, at `offset` from `row`, that lane r of 16 takes, as dwords
template <int BITS, int DP>
__device__ __forceinline__ void load_value(const uint8_t* base, uint32_t offset, int r, uint32_t* w) {
  const uint8_t* row = base + offset;
  if constexpr (BITS == 4) {
    const uint8_t* p = row + r * (DP / 32);
    if constexpr (DP == 32) w[0] = global_load<uint8_t>(p);
    else if constexpr (DP == 64) w[0] = global_load<uint16_t>(p);
    else if constexpr (DP == 96) w[0] = global_load<uint8_t>(p) | global_load<uint8_t>(p + 1) << 8 | global_load<uint8_t>(p + 2) << 16;
    else if constexpr (DP == 128) w[0] = global_load<uint32_t>(p);
    else if constexpr (DP == 192) {
      w[0] = global_load<uint16_t>(p) | global_load<uint16_t>(p + 2) << 16;
      w[1] = global_load<uint16_t>(p + 4);
    } else {
      const u32x2 v = global_load<u32x2>(p);
      w[0] = v[0], w[1] = v[1];
    }
  } else {
    if constexpr (DP == 32) w[0] = global_load<uint16_t>(row + 2 * r);
    else if constexpr (DP == 64) w[0] = global_load<uint32_t>(row + 4 * r);
    else if constexpr (DP == 96) w[0] = global_load<uint32_t>(row + 4 * r), w[1] = global_load<uint16_t>(row + 64 + 2 * r);
    else if constexpr (DP == 128) {
      const u32x2 v = global_load_nt<u32x2>(row + 8 * r);  // whole 128-byte lines
      w[0] = v[0], w[1] = v[1];
    } else if constexpr (DP == 192) {
      const u32x2 v = global_load<u32x2>(row + 8 * r);
      w[0] = v[0], w[1] = v[1], w[2] = global_load<uint32_t>(row + 128 + 4 * r);
    } else {
      const u32x4 v = global_load<u32x4>(row + 16 * r);
      w[0] = v[0], w[1] = v[1], w[2] = v[2], w[3] = v[3];
    }
  }
}

// the bytes of a key's row that its lane of group g takes
template <int BITS, int DP>
__device__ __forceinline__ void load_key(const uint8_t* base, uint32_t offset, int g, uint32_t* w) {
  const uint8_t* row = base + offset;
  if constexpr (BITS == 4) {
    const uint8_t* p = row + g * (DP / 8);
#pragma unroll
    for (int i = 0; i < DP / 32; i++) w[i] = global_load<uint32_t>(p + 4 * i);
  } else {
#pragma unroll
    for (int c = 0; c < DP / 64; c++) {
      const u32x4 v = global_load<u32x4>(row + 64 * c + 16 * g);
#pragma unroll
      for (int i = 0; i < 4; i++) w[4 * c + i] = v[i];
    }
    if constexpr (DP % 64 != 0) {
      const u32x2 v = global_load<u32x2>(row + DP / 64 * 64 + 8 * g);
      w[DP / 16 - 2] = v[0], w[DP / 16 - 1] = v[1];
    }
  }
}

// the first channel of depth group g in key product step k
template <int BITS, int DP>
__device__ __forceinline__ int key_channel(int k, int g) {
  if constexpr (BITS == 4) return 32 * k + 8 * g;
  else return k < DP / 64 * 2 ? 64 * (k >> 1) + 16 * g + 8 * (k & 1) : DP / 64 * 64 + 8 * g;
}

// Nibbles hold code + 8.  RAISED: as they are, in the high fraction bits of bf16
// numbers of 16 .. 31, code + 24: three operations for two codes, against five;
// what the 24 adds is taken away by the products (see `attend`).  Otherwise the
// code itself.
__device__ __forceinline__ uint32_t raised(uint32_t w, int nibble) {  // nibbles `nibble` and `nibble` + 4
  return ((nibble ? w >> (4 * nibble - 3) : w << 3) & 0x00780078u) | 0x41804180u;
}
constexpr uint32_t RAISE = 0xc1c0c1c0u;  // -24 twice

template <int BITS, bool RAISED>
__device__ __forceinline__ bf16x8 key_operand(const uint32_t* w, int k) {
  if constexpr (BITS == 8) {
    return bytes_bf16(w[2 * k], w[2 * k + 1]);
  } else {
    u32x4 out;
    const uint32_t x = w[k] ^ 0x88888888u;
#pragma unroll
    for (int e = 0; e < 4; e++) {  // nibbles e and e + 4
      if constexpr (RAISED) out[e] = raised(w[k], e);
      else out[e] = pack_bf16x2((float)((int32_t)(x << (28 - 4 * e)) >> 28), (float)((int32_t)(x << (12 - 4 * e)) >> 28));
    }
    return __builtin_bit_cast(bf16x8, out);
  }
}

// operand i of the value product from the eight keys' dwords (RAISED: of 16-bit halves of two keys each)
template <int BITS, bool RAISED, int W>
__device__ __forceinline__ bf16x8 value_operand(const uint32_t (&w)[8][W], int i) {
  u32x4 out;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if constexpr (BITS == 4 && RAISED) {
      out[e] = raised(w[2 * e + (i >> 2 & 1)][i >> 3], i & 3);
    } else {
      uint32_t a = w[2 * e][i * BITS / 32], b = w[2 * e + 1][i * BITS / 32];
      if constexpr (BITS == 4) a ^= 0x88888888u, b ^= 0x88888888u;
      const int s = 32 - BITS - i * BITS % 32;
      out[e] = pack_bf16x2((float)((int32_t)(a << s) >> (32 - BITS)), (float)((int32_t)(b << s) >> (32 - BITS)));
    }
  }
  return __builtin_bit_cast(bf16x8, out);
}

template <class T> __device__ __forceinline__ float element(const T* p, int64_t i);
template <> __device__ __forceinline__ float element<float>(const float* p, int64_t i) { return p[i]; }
template <> __device__ __forceinline__ float element<bf16_t>(const bf16_t* p, int64_t i) { return bf16_to_f32(p[i]); }

template <class T, int BITS, int DP, int TILE, int SPREAD, int BLOCKS = 1>
__global__ void __launch_bounds__(WAVES * 64) attend(AttendArgs a) {
  constexpr int KW = DP * BITS / 128;                             // dwords of a lane's share of a key row
  constexpr int VW = (DP * BITS / 128 + 3) / 4 < 1 ? 1 : (DP * BITS / 128 + 3) / 4;  // of a value row
  constexpr int G = BITS == 8 ? 1 : DP / 32;                      // scales of a row
  constexpr int KS = DP / 32, NV = DP / 16, QP = Parts<T>::Q, PP = Parts<T>::P;
  constexpr int ROWS = 16 / SPREAD;                               // rows of a tile of 16 columns
  constexpr bool RAISED = BITS == 4 && sizeof(T) == 2;
  constexpr int ROW = DP * BITS / 8;                              // bytes of a row
  constexpr int COPIES = SPREAD / BLOCKS, SIDE = 16 / BLOCKS;     // columns of a row and block, columns of a block
  constexpr int QN = BLOCKS > 1 ? BLOCKS : QP;
  static_assert(SPREAD == 1 || (TILE == 1 && COPIES >= PP), "a row's parts need a column each");
  static_assert(BLOCKS == 1 || QP == 1, "the queries of the other block's columns are zero");
  const int lane = threadIdx.x & 63, wave = uniform32(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int side = r / SIDE, part = r / ROWS % COPIES;  // the column's block, and which part of a probability it holds
  const int total = (int)gridDim.x, id = a.tiles > 1 ? xcd_remap(blockIdx.x, total) : (int)blockIdx.x;
  const int split = id % a.splits, tile = id / a.splits % a.tiles;
  const int64_t unit = id / a.splits / a.tiles, b = unit / a.kv_heads, head = unit % a.kv_heads;
  const int64_t given = a.counts ? a.counts[b] : a.fresh, count = given < a.fresh ? given : a.fresh;
  const int64_t first = a.start + (a.starts ? a.starts[b] : 0);
  const int64_t rows = a.fresh * a.group, row0 = (int64_t)tile * (ROWS * TILE);
  // the keys that a row sees; none where it is not a query
  auto sees = [&](int64_t row) -> int {
    const int64_t t = row / a.group, n = first + t + 1;
    return row < rows && t < count && n > 0 ? (int)(n < a.capacity ? n : a.capacity) : 0;
  };
  const int64_t last = row0 + ROWS * TILE < rows ? row0 + ROWS * TILE - 1 : rows - 1;
  const int64_t filled = count * a.group - 1;  // the last query's row
  const int end = filled < row0 ? 0 : sees(last < filled ? last : filled), least = sees(row0);
  int limit[TILE];
#pragma unroll
  for (int i = 0; i < TILE; i++) limit[i] = sees(row0 + i * ROWS + r % ROWS);

  // ---- queries: the columns' rows, PARTS of each depth
  bf16x8 q[TILE][KS][QN];
#pragma unroll
  for (int i = 0; i < TILE; i++) {
    const int64_t row = row0 + i * ROWS + r % ROWS, t = row / a.group;
    const T* p = (const T*)a.q + ((b * a.fresh + t) * a.heads + head * a.group + row % a.group) * a.dim;
#pragma unroll
    for (int k = 0; k < KS; k++) {
      const int d = key_channel<BITS, DP>(k, g);
      if constexpr (QP == 1) {
        u32x4 w = {0u, 0u, 0u, 0u};
        if (limit[i] && d < a.dim) {
          if (a.vector) {
            w = global_load<u32x4>(p + d);
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
              if (d + e < a.dim) w[e >> 1] |= (uint32_t)p[d + e] << (16 * (e & 1));
          }
        }
#pragma unroll
        for (int c = 0; c < QN; c++) {
          const u32x4 none = {0u, 0u, 0u, 0u};
          q[i][k][c] = __builtin_bit_cast(bf16x8, side == c ? w : none);
        }
      } else {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = limit[i] && d + e < a.dim ? element(p, d + e) : 0.f;
        split_bf16<QP>(v, q[i][k]);
      }
    }
  }

  // what the raised keys add to a group's products, taken off in fp32: some six times a code's size, whose
  // rounding stays far below a bf16 output's
  f32x4 drop[TILE][RAISED ? G : 1];
  if constexpr (RAISED) {
    const u32x4 raise = {RAISE, RAISE, RAISE, RAISE};
#pragma unroll
    for (int i = 0; i < TILE; i++)
#pragma unroll
      for (int k = 0; k < KS; k++) {
        drop[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < QN; c++)
          drop[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, raise), q[i][k][c], drop[i][k], 0, 0, 0);
      }
  }

  f32x4 acc[TILE][NV];
  float top[TILE], sum[TILE];
#pragma unroll
  for (int i = 0; i < TILE; i++) {
    top[i] = LOWEST, sum[i] = 0.f;
#pragma unroll
    for (int n = 0; n < NV; n++) acc[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // ---- this workgroup's keys, BLOCKS blocks of 32 per wave at a time
  constexpr int STEP = BLOCK * BLOCKS;
  const int share = ((end + a.splits - 1) / a.splits + STEP * WAVES - 1) / (STEP * WAVES) * (STEP * WAVES);
  const int from = split * share, to = from + share < end ? from + share : end;
  const int64_t base = unit * a.capacity;
  const uint8_t* K = a.codes[0] + base * ROW;
  const uint8_t* V = a.codes[1] + base * ROW;
  const bf16_t* KSC = a.scales[0] + base * G;
  const bf16_t* VSC = a.scales[1] + base * G;
  for (int s0 = from + wave * STEP; s0 < to; s0 += WAVES * STEP) {
    uint32_t kw[BLOCKS][2][KW], vw[BLOCKS][8][VW], ks[2][2 * G], vs[2][2 * G];
    const bf16_t* key_scales = KSC + (int64_t)s0 * G;
    const bf16_t* value_scales = VSC + (int64_t)s0 * G;
    // the last block may stand alone: then it is taken twice, and no row sees the second's keys (end <= s0 + 32)
    const bool both = s0 + BLOCK < to;
    const int own = both ? BLOCK * side : 0;
#pragma unroll
    for (int c = 0; c < BLOCKS; c++) {
      const uint8_t* key_rows = K + (int64_t)(s0 + (c && both ? BLOCK : 0)) * ROW;
#pragma unroll
      for (int u = 0; u < 2; u++) load_key<BITS, DP>(key_rows, (uint32_t)((16 * u + r) * ROW), g, kw[c][u]);
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int n = 0; n < 2 * G; n++) {
        ks[u][n] = global_load<uint32_t>(key_scales + (uint32_t)((own + 16 * u + 4 * g) * G + 2 * n));
        vs[u][n] = global_load<uint32_t>(value_scales + (uint32_t)((own + 16 * u + 4 * g) * G + 2 * n));
      }
    }
#pragma unroll
    for (int c = 0; c < BLOCKS; c++) {
      const uint8_t* value_rows = V + (int64_t)(s0 + (c && both ? BLOCK : 0)) * ROW;
#pragma unroll
      for (int j = 0; j < 8; j++)
        load_value<BITS, DP>(value_rows, (uint32_t)((16 * (j >> 2) + 4 * g + (j & 3)) * ROW), r, vw[c][j]);
    }
    __builtin_amdgcn_sched_barrier(0);  // all of a block's loads are in flight before the first is waited for
    if constexpr (RAISED) {  // the halves of two keys' dwords beside each other
#pragma unroll
      for (int c = 0; c < BLOCKS; c++)
#pragma unroll
        for (int j = 0; j < 8; j += 2)
#pragma unroll
          for (int n = 0; n < VW; n++) {
            const uint32_t lo = __builtin_amdgcn_perm(vw[c][j + 1][n], vw[c][j][n], 0x05040100u);
            vw[c][j + 1][n] = __builtin_amdgcn_perm(vw[c][j + 1][n], vw[c][j][n], 0x07060302u);
            vw[c][j][n] = lo;
          }
    }

    // scores, before the factor that makes them powers of two
    f32x4 score[TILE][2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      f32x4 dot[TILE][G];
#pragma unroll
      for (int i = 0; i < TILE; i++)
#pragma unroll
        for (int n = 0; n < G; n++) {
          if constexpr (RAISED) dot[i][n] = drop[i][n];
          else dot[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
      for (int ck = 0; ck < BLOCKS * KS; ck++) {
        const int c = ck / KS, k = ck % KS;
        const bf16x8 key = key_operand<BITS, RAISED>(kw[c][u], k);
#pragma unroll
        for (int i = 0; i < TILE; i++)
#pragma unroll
          for (int n = BLOCKS > 1 ? c : 0; n < (BLOCKS > 1 ? c + 1 : QP); n++)
            dot[i][G == 1 ? 0 : k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key, q[i][k][n], dot[i][G == 1 ? 0 : k], 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 4; e++) {
#pragma unroll
        for (int i = 0; i < TILE; i++) {
          float x = 0.f;
#pragma unroll
          for (int n = 0; n < G; n++) {
            const float s = scale_at(ks[u], e * G + n);
            x = G == 1 ? dot[i][0][e] * s : __builtin_fmaf(dot[i][n][e], s, x);
          }
          score[i][u][e] = x;
        }
      }
    }
    if (s0 + STEP > least) {  // the block has keys that some row does not see
#pragma unroll
      for (int i = 0; i < TILE; i++)
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (s0 + BLOCK * side + 16 * u + 4 * g + e >= limit[i]) score[i][u][e] = -INFINITY;
    }
    // probabilities relative to the row's running maximum
    float p[TILE][8];
#pragma unroll
    for (int i = 0; i < TILE; i++) {
      float m = fmaxf(fmaxf(fmaxf(score[i][0][0], score[i][0][1]), fmaxf(score[i][0][2], score[i][0][3])),
                      fmaxf(fmaxf(score[i][1][0], score[i][1][1]), fmaxf(score[i][1][2], score[i][1][3])));
      m *= a.scale;
      if (__any(m > top[i] + RISE)) {
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(fmaxf(m, __shfl_xor(m, 32)), top[i]);
        const float fade = __builtin_amdgcn_exp2f(top[i] - m);
        top[i] = m;
        sum[i] *= fade;
#pragma unroll
        for (int n = 0; n < NV; n++) acc[i][n] *= fade;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        p[i][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[i][j >> 2][j & 3], a.scale, -top[i]));
        sum[i] += p[i][j];
      }
    }
    // values
#pragma unroll
    for (int n = 0; n < G; n++) {
      bf16x8 weights[TILE][SPREAD > 1 ? 1 : PP];
#pragma unroll
      for (int i = 0; i < TILE; i++) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = p[i][j] * scale_at(vs[j >> 2], (j & 3) * G + n);
        if (s0 + STEP > least) {  // 0 for what the row does not see, whatever its scale
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (s0 + BLOCK * side + 16 * (j >> 2) + 4 * g + (j & 3) >= limit[i]) x[j] = 0.f;
        }
        if constexpr (SPREAD > 1) {  // the column's part alone
          u32x4 w;
#pragma unroll
          for (int n2 = 0; n2 < PP; n2++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              w[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
              if (n2 + 1 < PP) {
                const float more = part > n2 ? 1.f : 0.f;
                x[2 * e] = __builtin_fmaf(-more, __uint_as_float(w[e] << 16), x[2 * e]);
                x[2 * e + 1] = __builtin_fmaf(-more, __uint_as_float(w[e] & 0xffff0000u), x[2 * e + 1]);
              }
            }
          }
          if (COPIES > PP && part >= PP) w = u32x4{0u, 0u, 0u, 0u};  // more columns than parts
          weights[i][0] = __builtin_bit_cast(bf16x8, w);
        } else {
          split_bf16<PP>(x, weights[i]);
        }
      }
      bf16x8 sided[BLOCKS];  // the weights of a block's columns, 0 in the other's
      if constexpr (BLOCKS > 1) {
        const u32x4 none = {0u, 0u, 0u, 0u}, w = __builtin_bit_cast(u32x4, weights[0][0]);
#pragma unroll
        for (int c = 0; c < BLOCKS; c++) sided[c] = __builtin_bit_cast(bf16x8, side == c ? w : none);
      }
#pragma unroll
      for (int v = n * (NV / G); v < (n + 1) * (NV / G); v++) {
#pragma unroll
        for (int c = 0; c < BLOCKS; c++) {
          const bf16x8 value = value_operand<BITS, RAISED, VW>(vw[c], v);
#pragma unroll
          for (int i = 0; i < TILE; i++)
#pragma unroll
            for (int n2 = 0; n2 < (SPREAD > 1 ? 1 : PP); n2++)
              acc[i][v] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value, BLOCKS > 1 ? sided[c] : weights[i][n2], acc[i][v], 0, 0, 0);
        }
        if constexpr (RAISED) {  // block by block: the sums never hold more than a block's excess
          const u32x4 raise = {RAISE, RAISE, RAISE, RAISE};
#pragma unroll
          for (int i = 0; i < TILE; i++)
#pragma unroll
            for (int n2 = 0; n2 < (SPREAD > 1 ? 1 : PP); n2++)
              acc[i][v] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, raise), weights[i][n2], acc[i][v], 0, 0, 0);
        }
      }
    }
  }

  // ---- the waves' softmaxes joined, two operands' rows of 16 channels at a time
  constexpr int CHUNK = 2;
  __shared__ float tops[WAVES][16], sums[WAVES][16], stage[WAVES][CHUNK][16][17];
#pragma unroll
  for (int i = 0; i < TILE; i++) {
    sum[i] += __shfl_xor(sum[i], 16);
    sum[i] += __shfl_xor(sum[i], 32);
    __syncthreads();
    if (g == 0) tops[wave][r] = top[i], sums[wave][r] = sum[i];
    __syncthreads();
    float most = LOWEST;
#pragma unroll
    for (int c = 0; c < BLOCKS; c++)
#pragma unroll
      for (int w = 0; w < WAVES; w++) most = fmaxf(most, tops[w][r % ROWS + c * SIDE]);
    const float fade = __builtin_amdgcn_exp2f(top[i] - most);
    // thread c % 16 = row r' of the products, c / 16 = column
    const int channel_row = threadIdx.x & 15, column = threadIdx.x >> 4, row = column % ROWS;
    float whole = 0.f, high = LOWEST;
#pragma unroll
    for (int c = 0; c < BLOCKS; c++)
#pragma unroll
      for (int w = 0; w < WAVES; w++) high = fmaxf(high, tops[w][row + c * SIDE]);
#pragma unroll
    for (int c = 0; c < BLOCKS; c++)
#pragma unroll
      for (int w = 0; w < WAVES; w++)
        whole += sums[w][row + c * SIDE] * __builtin_amdgcn_exp2f(tops[w][row + c * SIDE] - high);
    const int64_t at = row0 + i * ROWS + row, t = at / a.group;
    const bool writes = column < ROWS && at < rows;
    if (sees(at) == 0) whole = 0.f;  // not a query, or one without keys: zero
    T* out = (T*)a.out + ((b * a.fresh + t) * a.heads + head * a.group + at % a.group) * a.dim;
    const int64_t slot = ((int64_t)(unit * a.tiles + tile) * a.splits + split) * (ROWS * TILE) + i * ROWS + row;
    if (a.splits > 1 && writes && channel_row == 0) {
      a.stats[2 * slot] = high;
      a.stats[2 * slot + 1] = whole;
    }
#pragma unroll
    for (int n0 = 0; n0 < NV; n0 += CHUNK) {
#pragma unroll
      for (int n = 0; n < CHUNK; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) stage[wave][n][r][4 * g + e] = acc[i][n0 + n][e] * fade;
      __syncthreads();
      if (writes) {
#pragma unroll
        for (int n = 0; n < CHUNK; n++) {
          float v = 0.f;
#pragma unroll
          for (int c = 0; c < SPREAD; c++)
#pragma unroll
            for (int w = 0; w < WAVES; w++) v += stage[w][n][row + c * ROWS][channel_row];
          const int d = value_channel<BITS, DP>(n0 + n, channel_row);
          if (a.splits > 1) {
            a.part[slot * DP + d] = v;
          } else if (d < a.dim) {
            v = whole == 0.f ? 0.f : v / whole;
            if constexpr (sizeof(T) == 2) out[d] = f32_to_bf16(v);
            else out[d] = v;
          }
        }
      }
      __syncthreads();
    }
  }
}

// The ranges of split rows joined: a wave per row.  Bound by latency (a chain of
// two loads): the lanes hold a range's maximum and weight each.
template <class T, int DP>
__global__ void __launch_bounds__(64) attend_join(AttendArgs a, int tile_rows) {
  constexpr int N = (DP + 63) / 64, RANGES = 256 / 64;
  __shared__ float fades[256];
  const int lane = threadIdx.x;
  const uint32_t at = blockIdx.x, h = at % (uint32_t)a.heads, bt = at / (uint32_t)a.heads, t = bt % (uint32_t)a.fresh;
  const uint32_t b = bt / (uint32_t)a.fresh, row = t * a.group + h % a.group;
  const int64_t unit = (int64_t)b * a.kv_heads + h / a.group;
  const int64_t slot = (unit * a.tiles + row / tile_rows) * a.splits * tile_rows + row % tile_rows;
  float top[RANGES], weight[RANGES], most = LOWEST, whole = 0.f;
#pragma unroll
  for (int i = 0; i < RANGES; i++) {
    const int s = lane + 64 * i;
    u32x2 w = {__float_as_uint(LOWEST), 0u};
    if (s < a.splits) w = global_load<u32x2>(a.stats + 2 * (slot + (int64_t)s * tile_rows));
    top[i] = __uint_as_float(w[0]), weight[i] = __uint_as_float(w[1]);
    most = fmaxf(most, top[i]);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
#pragma unroll
  for (int i = 0; i < RANGES; i++) {
    const float fade = __builtin_amdgcn_exp2f(top[i] - most);
    fades[lane + 64 * i] = fade;
    whole += weight[i] * fade;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) whole += __shfl_xor(whole, o);
  __syncthreads();
  float v[N] = {};
#pragma unroll 8
  for (int s = 0; s < a.splits; s++) {
    const float* part = a.part + (slot + (int64_t)s * tile_rows) * DP;
    const float fade = fades[s];
#pragma unroll
    for (int n = 0; n < N; n++)
      if (DP % 64 == 0 || lane + 64 * n < DP) v[n] = __builtin_fmaf(global_load<float>(part + lane + 64 * n), fade, v[n]);
  }
  T* out = (T*)a.out + (int64_t)at * a.dim;
#pragma unroll
  for (int n = 0; n < N; n++) {
    const int d = lane + 64 * n;
    if (d >= a.dim) continue;
    const float x = whole == 0.f ? 0.f : v[n] / whole;
    if constexpr (sizeof(T) == 2) out[d] = f32_to_bf16(x);
    else out[d] = x;
  }
}

template <class T, int BITS, int DP>
int attend_width(const AttendArgs& a, const AttendPlan& p, hipStream_t stream) {
  const dim3 grid((unsigned)(a.units * p.tiles * p.splits)), block(WAVES * 64);
  if (p.spread == 4) {
    hipLaunchKernelGGL((attend<T, BITS, DP, 1, 4, blocks_of(sizeof(T), BITS, DP)>), grid, block, 0, stream, a);
  } else if (p.spread == 2) {
    if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((attend<T, BITS, DP, 1, 2>), grid, block, 0, stream, a);
  } else if constexpr (one_tile(sizeof(T), BITS, DP)) {
    hipLaunchKernelGGL((attend<T, BITS, DP, 1, 1>), grid, block, 0, stream, a);
  } else {
    if constexpr (sizeof(T) == 2 && DP <= 128) {
      if (p.tile == 4) hipLaunchKernelGGL((attend<T, BITS, DP, 4, 1>), grid, block, 0, stream, a);
    }
    if (p.tile == 2) hipLaunchKernelGGL((attend<T, BITS, DP, 2, 1>), grid, block, 0, stream, a);
  }
  if (p.splits > 1)
    hipLaunchKernelGGL((attend_join<T, DP>), dim3((unsigned)(a.units / a.kv_heads * a.fresh * a.heads)), dim3(64), 0, stream, a,
                       p.rows);
  return (int)hipGetLastError();
}

template <class T>
int attend_type(const AttendArgs& a, const AttendPlan& p, int bits, hipStream_t stream) {
  auto width = [&](auto code_bits) {
    constexpr int BITS = decltype(code_bits)::value;
    switch (p.pitch) {
      case 32: return attend_width<T, BITS, 32>(a, p, stream);
      case 64: return attend_width<T, BITS, 64>(a, p, stream);
      case 96: return attend_width<T, BITS, 96>(a, p, stream);
      case 128: return attend_width<T, BITS, 128>(a, p, stream);
      case 192: return attend_width<T, BITS, 192>(a, p, stream);
      default: return attend_width<T, BITS, 256>(a, p, stream);
    }
  };
  return bits == 8 ? width(std::integral_constant<int, 8>()) : width(std::integral_constant<int, 4>());
}

}  // namespace

// one translation unit for each storage type
namespace qa {
int attend_bf16(const void* args, const void* plan, int bits, hipStream_t stream);
int attend_fp32(const void* args, const void* plan, int bits, hipStream_t stream);
}  // namespace qa
