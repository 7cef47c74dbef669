// Attention of sequences of different lengths that lie one behind the other in
// one matrix of tokens: C ABI `qutai_amd_attention_packed_fwd`, `_bwd`, `_rows`,
// `_workspace`.
//
//   forward:  S = scale Q K^T over a sequence's own (causal: no later) keys,
//             O = softmax(S) V, lse = log sum exp S
//   backward: P = exp(S - lse), dV = P^T dO, dP = dO V^T, delta = rowsum(dO O),
//             dS = P (dP - delta), dQ = scale dS K, dK = scale dS^T Q.
//
// The caller's tile tables say which rows of which sequence a workgroup takes, in
// the order in which the workgroups start; every tile lies in one sequence, so
// padding costs no work and no mask but a sequence's own end is needed.  bf16 heads of
// up to 128 channels take the kernels of attention_packed.h, fp32 and wider heads those
// that keep fp32 values in bf16 parts (attention_mma.h), rows that are not whole
// 16-byte chunks, fp32 ones wider than 128 channels and sequences of a few tokens one wave per
// row (attention_rows.h; 3000 tokens of up to 500, 16 heads over 4, fp32 of 160: 1340, 1160 and
// 2150 us).
//
// fp32: 2999 tokens of 34 sequences of 2 to 500, every token sees its whole sequence, 12
// heads of 80: forward 54 us, dQ 71, dK and dV 91, 10.3 GFLOP in all (the six products of
// the parts run at 290 TFLOP/s): a wave has its SIMD to itself (350 registers and more),
// and its reads, products and vector instructions follow each other.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "attention_packed.h"

namespace {

constexpr int64_t MMA_ROWS = 128;  // queries or keys of a workgroup of attention_mma.h's kernels
constexpr int WAVES = 4;           // of a workgroup of attention_packed.h's query kernels

template <class T>
__global__ void __launch_bounds__(GEN_WAVES * 64) packed_fwd_rows(AttnPackedArgs p) {
  int b, h, blk;
  place_queries<T, GEN_WAVES>(p, b, h, blk);
  const int t = blk * GEN_WAVES + uniform32(threadIdx.x >> 6);
  if (t < p.time) fwd_row<T>(p, b, h, t, threadIdx.x & 63);
}
template <class T>
__global__ void __launch_bounds__(GEN_WAVES * 64) packed_bwd_q_rows(AttnPackedArgs p) {
  int b, h, blk;
  place_queries<T, GEN_WAVES>(p, b, h, blk);
  const int t = blk * GEN_WAVES + uniform32(threadIdx.x >> 6);
  if (t < p.time) bwd_q_row<T>(p, b, h, t, threadIdx.x & 63);
}
template <class T>
__global__ void __launch_bounds__(GEN_WAVES * 64) packed_bwd_kv_rows(AttnPackedArgs p) {
  int b, kvh, blk, gsel;
  place_keys<T, GEN_WAVES>(p, 1, b, kvh, blk, gsel);
  const int t = blk * GEN_WAVES + uniform32(threadIdx.x >> 6);
  if (t < p.time) bwd_kv_row<T>(p, b, kvh, t, threadIdx.x & 63, 0, (int)(p.heads / p.kv_heads));
}

enum Pass { FORWARD, QUERIES, KEYS };

// How a workgroup of the key pass is cut: waves of 32 keys each, and sets of them
// that share the group's query heads.
struct KeyShape {
  int waves, sets;
};

// `tiles` bounds the key tiles from above (of 64 rows, for each kv head).  Many of
// them: as many workgroups as fit a CU (registers allow two waves of each SIMD).  Few:
// a workgroup is a CU's only one, four sets of waves take a head each, and the longest
// tile ends in a quarter of the time.  Measured, us: 16384 tokens of up to 1024, 16
// heads over 4 of 64, {2, 2} 76, {4, 2} 92-99, {2, 4} 114, {4, 1} 155; one of 2000, 8
// over 2 of 64, {2, 2} 103, {2, 4} 76; 16000 of up to 6000, 32 over 8 of 128, {4, 1}
// 1580, {2, 2} 2146 (its sums spill to the accumulation registers); 500 at most, 193 and
// 247; 16384 of up to 1024, 16 over 4 of 80, {4, 1} 165, {2, 2} 116, 12 over 12 of 96, {4, 1}
// 102, {2, 1} 99; 8000 of up to 2000, 16 over 4 of 96, {2, 2} 172, {2, 4} 136; 8000 of up
// to 8, 16 over 4 of 64, {2, 2} 157, {2, 4} 335.
// Short sequences (ONLY kernels): tiles of 64 rows, which hold one; 16000 of up to 64, 32
// heads over 8 of 128, {2, 1} 173; 8000, 16 over 4 of 96, {2, 1} 29, {2, 2} 40 to 77 (it
// spills); 16384, 16 over 4 of 64, {2, 2} 60.
KeyShape key_shape(int64_t heads, int64_t kv_heads, int64_t dim, int64_t tiles, int64_t longest) {
  const int64_t group = heads / kv_heads;
  if (longest <= FINE) return dim <= 64 && group % 2 == 0 ? KeyShape{2, 2} : KeyShape{2, 1};
  const bool few = tiles * kv_heads < 2 * cu_count() * (dim > 64 ? 2 : 1);
  if (few && group % 4 == 0) return {2, 4};
  if (dim <= 96) return group % 2 == 0 ? KeyShape{2, 2} : KeyShape{2, 1};
  return few && group % 2 == 0 ? KeyShape{4, 2} : KeyShape{4, 1};
}

int64_t key_tiles_of(int64_t tokens, int64_t sequences) { return tokens / 64 + std::min(sequences, tokens); }

template <int DP>
void launch_packed(Pass pass, const AttnPackedArgs& a, unsigned blocks, KeyShape shape, bool only, hipStream_t stream) {
  if (pass != KEYS) {
    const dim3 block(WAVES * 64);
    if (pass == FORWARD) hipLaunchKernelGGL((packed_fwd<DP, WAVES, DP <= 64 ? 64 : 32>), dim3(blocks), block, 0, stream, a);
    else hipLaunchKernelGGL((packed_bwd_dq<DP, WAVES>), dim3(blocks), block, 0, stream, a);
    return;
  }
  const auto [waves, sets] = shape;
  const dim3 block(waves * sets * 64);
  if (only) {
    constexpr int MOST = DP <= 64 ? 2 : 1;
    if (sets == MOST) hipLaunchKernelGGL((packed_bwd_dkv<DP, 2, MOST, true>), dim3(blocks), block, 0, stream, a);
    else hipLaunchKernelGGL((packed_bwd_dkv<DP, 2, 1, true>), dim3(blocks), block, 0, stream, a);
  } else if (sets == 4) {
    hipLaunchKernelGGL((packed_bwd_dkv<DP, 2, 4>), dim3(blocks), block, 0, stream, a);
  } else if constexpr (DP <= 96) {
    if (sets == 2) hipLaunchKernelGGL((packed_bwd_dkv<DP, 2, 2>), dim3(blocks), block, 0, stream, a);
    else hipLaunchKernelGGL((packed_bwd_dkv<DP, 2, 1>), dim3(blocks), block, 0, stream, a);
  } else {
    if (sets == 2) hipLaunchKernelGGL((packed_bwd_dkv<DP, 4, 2>), dim3(blocks), block, 0, stream, a);
    else hipLaunchKernelGGL((packed_bwd_dkv<DP, 4, 1>), dim3(blocks), block, 0, stream, a);
  }
}

template <bool F32, int DP>
void launch_mma(Pass pass, const AttnPackedArgs& a, unsigned blocks, hipStream_t stream) {
  const dim3 grid(blocks), block(256);
  if (pass == FORWARD) hipLaunchKernelGGL((attention_fwd_mma<F32, DP, AttnPackedArgs>), grid, block, 0, stream, a);
  else if (pass == QUERIES)
    hipLaunchKernelGGL((attention_bwd_dq_mma<F32, DP, AttnPackedArgs>), grid, block, 0, stream, a);
  else if constexpr (DP > 128) {
    hipLaunchKernelGGL((attention_bwd_dkv_mma<F32, DP, KEYS_DV, AttnPackedArgs>), grid, block, 0, stream, a);
    hipLaunchKernelGGL((attention_bwd_dkv_mma<F32, DP, KEYS_DK, AttnPackedArgs>), grid, block, 0, stream, a);
  } else {
    hipLaunchKernelGGL((attention_bwd_dkv_mma<F32, DP, KEYS_BOTH, AttnPackedArgs>), grid, block, 0, stream, a);
  }
}

template <class T>
void launch_rows(Pass pass, const AttnPackedArgs& a, unsigned blocks, hipStream_t stream) {
  const dim3 grid(blocks), block(GEN_WAVES * 64);
  if (pass == FORWARD) hipLaunchKernelGGL(packed_fwd_rows<T>, grid, block, 0, stream, a);
  else if (pass == QUERIES) hipLaunchKernelGGL(packed_bwd_q_rows<T>, grid, block, 0, stream, a);
  else hipLaunchKernelGGL(packed_bwd_kv_rows<T>, grid, block, 0, stream, a);
}

// Whether the matrix kernels take rows of this type and width (of whole 16-byte chunks).
bool mma_fits(int dtype, int64_t dim) { return dtype == BF16 ? dim % 8 == 0 && dim <= 256 : dim % 4 == 0 && dim <= 128; }

bool packed_fits(int dtype, int64_t dim) { return dtype == BF16 && dim % 8 == 0 && dim <= 128; }

// Workgroups of a tile: heads of its side, less those that share one.
int64_t groups_of(Pass pass, int dtype, int64_t heads, int64_t kv_heads, int64_t dim, int64_t rows) {
  if (pass == KEYS) return kv_heads;
  return rows != GEN_WAVES && packed_fits(dtype, dim) ? heads / packed_heads(heads, kv_heads, WAVES) : heads;
}

// Query heads of a group that take workgroups of their own in the key pass of
// attention_mma.h's kernels, whose partial sums a kernel of its own adds up: all of
// them with fewer workgroups than the GPU holds at once (two for a CU), else 1.  us,
// side by side (with the sum) and one after the other: fp32, one sequence of 4000, 8
// heads over 2 of 64, 412 and 1530; 4000 tokens of up to 1000, 16 over 4 of 64, 126 and
// 400, 8000 with heads of 32, 96 and 238; bf16 of 256, 564 and 1134; with half as many
// tiles again as the bound, 16384 of up to 1024, 16 over 4 of 64, 414 and 440, 8 over 4
// of 96, 304 and 308, and with three times as many, 16 over 8 of 64, 424 and 375.
int64_t heads_apart(int dtype, int64_t tokens, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t dim, int64_t rows) {
  if (rows == GEN_WAVES || packed_fits(dtype, dim)) return 1;
  return (tokens / MMA_ROWS + std::min(sequences, tokens)) * kv_heads < 2 * cu_count() ? heads / kv_heads : 1;
}

// dK = scale * sum_g part_k[g], dV = sum_g part_v[g] (g in order) of 4 channels a lane.
template <class T>
__global__ void __launch_bounds__(256) packed_dkv_sum(AttnPackedArgs p, int64_t tokens, int group) {
  constexpr bool F32 = sizeof(T) == 4;
  const int64_t chunks = p.kv_heads * p.dim / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x, t = i / chunks, at = i % chunks * 4;
  if (t >= tokens) return;
  f32x4 sk = global_load<f32x4>(p.part_k + 4 * i), sv = global_load<f32x4>(p.part_v + 4 * i);
  for (int g = 1; g < group; g++) {
    sk += global_load<f32x4>(p.part_k + g * p.part_stride + 4 * i);
    sv += global_load<f32x4>(p.part_v + g * p.part_stride + 4 * i);
  }
  put4<F32>(p.dk, t * p.dkt + at, sk * p.scale);
  put4<F32>(p.dv, t * p.dvt + at, sv);
}

// Rows of a tile of the matrix kernels.
int64_t rows_of(Pass pass, int dtype, int64_t heads, int64_t kv_heads, int64_t dim, int64_t key_tiles, int64_t longest) {
  if (!packed_fits(dtype, dim)) return MMA_ROWS;
  if (pass == KEYS) return 32 * key_shape(heads, kv_heads, dim, key_tiles, longest).waves;
  return WAVES * 32 / packed_heads(heads, kv_heads, WAVES);
}

// One pass over the tiles of `rows` rows each.
hipError_t launch(Pass pass, int dtype, AttnPackedArgs a, int64_t key_tiles, int64_t longest, const int64_t* tiles,
                  int64_t count, int64_t rows, hipStream_t stream) {
  if (!count) return hipSuccess;
  a.tiles = tiles;
  a.lengths = tiles + count;
  a.pack = packed_heads(a.heads, a.kv_heads, WAVES);
  const int64_t apart = pass == KEYS && a.split ? a.heads / a.kv_heads : 1;
  const unsigned n = (unsigned)(count * groups_of(pass, dtype, a.heads, a.kv_heads, a.dim, rows) * apart);
  if (rows == GEN_WAVES) {
    if (dtype == BF16) launch_rows<bf16_t>(pass, a, n, stream);
    else launch_rows<float>(pass, a, n, stream);
  } else if (dtype == BF16) {
    const KeyShape shape = key_shape(a.heads, a.kv_heads, a.dim, key_tiles, longest);
    if (a.dim <= 32) launch_packed<32>(pass, a, n, shape, longest <= FINE, stream);
    else if (a.dim <= 64) launch_packed<64>(pass, a, n, shape, longest <= FINE, stream);
    else if (a.dim <= 96) launch_packed<96>(pass, a, n, shape, longest <= FINE, stream);
    else if (a.dim <= 128) launch_packed<128>(pass, a, n, shape, longest <= FINE, stream);
    else launch_mma<false, 256>(pass, a, n, stream);
  } else {
    if (a.dim <= 32) launch_mma<true, 32>(pass, a, n, stream);
    else if (a.dim <= 64) launch_mma<true, 64>(pass, a, n, stream);
    else if (a.dim <= 96) launch_mma<true, 96>(pass, a, n, stream);
    else launch_mma<true, 128>(pass, a, n, stream);
  }
  return hipGetLastError();
}

// What forward and backward share: sizes, scale, pitches.  rows: of a tile.
int set_packed(AttnPackedArgs& a, int64_t tokens, int64_t sequences, int64_t longest, int64_t heads, int64_t kv_heads, int64_t dim,
               int64_t q_row, int64_t k_row, int64_t v_row, int dtype, double scale, int causal,
               std::initializer_list<std::pair<Pass, int64_t>> tiles) {
  if ((dtype != BF16 && dtype != F32) || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > 1 << 16) return QA_EINVAL;
  if (tokens < 0 || tokens >= 1ll << 31 || sequences < 0 || longest < 0) return QA_EINVAL;
  if (dim <= 0 || dim > 256 || !(scale > 0.0) || scale > 1e30) return QA_EINVAL;
  if (q_row < heads * dim || k_row < kv_heads * dim || v_row < kv_heads * dim) return QA_EINVAL;
  if (std::max({q_row, k_row, v_row, heads * dim}) > 1 << 22) return QA_EINVAL;  // 64 rows within a buffer descriptor
  for (const auto& [pass, rows] : tiles) {
    if (rows == GEN_WAVES) continue;
    if (rows != rows_of(pass, dtype, heads, kv_heads, dim, key_tiles_of(tokens, sequences), longest) || !mma_fits(dtype, dim) ||
        scale < 0x1p-50)
      return QA_EINVAL;
  }
  a.batch = 1;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dim = dim;
  a.qh = a.kh = dim;
  a.qt = q_row;
  a.kt = k_row;
  a.vt = v_row;
  a.ot = heads * dim;
  a.lh = 1;
  a.lt = heads;
  a.scale = (float)scale;
  const double log2 = scale * 1.4426950408889634 * (dtype == F32 ? 0x1p-48 : 1.0);
  a.scale_log2 = (float)log2;
  a.scale_log2_lo = (float)(log2 - (double)a.scale_log2);
  a.causal = causal ? 1 : 0;
  return QA_OK;
}

bool whole(std::initializer_list<const void*> pointers, std::initializer_list<int64_t> pitches, int dtype) {
  for (int64_t pitch : pitches)
    if (pitch * (dtype == F32 ? 4 : 2) % 16) return false;
  return aligned16(pointers);
}

// Whether a launch can hold a pass's workgroups, of 512 threads at most (`apart`: heads of a
// group that take workgroups of their own).
bool grid_fits(int64_t tiles, int64_t groups, int64_t apart = 1) {
  return tiles >= 0 && tiles <= ((1ll << 23) - 1) / (groups * apart);
}

}  // namespace

extern "C" {

int64_t qutai_amd_attention_packed_rows(int64_t tokens, int64_t sequences, int64_t longest, int64_t heads, int64_t kv_heads,
                                        int64_t dim, int dtype, int aligned, double scale, int pass) {
  if ((dtype != BF16 && dtype != F32) || dim <= 0 || dim > 256 || pass < 0 || pass > 2 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads || tokens < 0 || tokens >= 1ll << 31 || sequences < 0 || longest < 0)
    return 0;
  if (!aligned || !mma_fits(dtype, dim) || scale < 0x1p-50) return GEN_WAVES;
  // Tiles of sequences of a few tokens are mostly empty.  8000 tokens, us, tiles and one
  // wave per row: bf16, 16 heads over 4 of 64, sequences of up to 4, forward 73 and 80; of
  // up to 8, forward 49 and 91, dQ 58 and 104, dK and dV 157 and 70; fp32 of up to 8, 371 and
  // 89, 582 and 101, 646 and 69, of up to 16 194 and 117, 307 and 130, 332 and 104, of up to
  // 32 82 and 202, 132 and 217, 144 and 197.
  const int64_t few = packed_fits(dtype, dim) ? (pass == KEYS ? 8 : 0) : 20;
  if (longest <= few) return GEN_WAVES;
  return rows_of((Pass)pass, dtype, heads, kv_heads, dim, key_tiles_of(tokens, sequences), longest);
}

size_t qutai_amd_attention_packed_workspace(int64_t tokens, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t dim,
                                            int dtype, int64_t key_rows) {
  if ((dtype != BF16 && dtype != F32) || dim <= 0 || dim > 256 || heads <= 0 || kv_heads <= 0 || heads % kv_heads ||
      heads > 1 << 16 || tokens < 0 || tokens >= 1ll << 31 || sequences < 0)
    return 0;
  const int64_t apart = heads_apart(dtype, tokens, sequences, heads, kv_heads, dim, key_rows);
  return apart == 1 ? 0 : (size_t)(2 * apart * tokens * kv_heads * dim) * sizeof(float);
}

int qutai_amd_attention_packed_fwd(const void* q, const void* k, const void* v, void* out, float* lse, void* rest,
                                   const int64_t* tiles, int64_t tile_count, int64_t tile_rows, int64_t tokens, int64_t sequences,
                                   int64_t longest, int64_t heads, int64_t kv_heads, int64_t dim, int64_t q_row, int64_t k_row,
                                   int64_t v_row, int dtype, double scale, int causal, void* stream) {
  AttnPackedArgs a = {};
  const int status = set_packed(a, tokens, sequences, longest, heads, kv_heads, dim, q_row, k_row, v_row, dtype, scale, causal,
                                {{FORWARD, tile_rows}});
  if (status != QA_OK) return status;
  if (!grid_fits(tile_count, groups_of(FORWARD, dtype, heads, kv_heads, dim, tile_rows))) return QA_EINVAL;
  if (rest && (tile_rows == GEN_WAVES || !packed_fits(dtype, dim))) return QA_EINVAL;
  if (!tile_count) return QA_OK;
  if (!q || !k || !v || !out || !lse || !tiles) return QA_EINVAL;
  if (tile_rows != GEN_WAVES && !whole({q, k, v, out, rest ? rest : out}, {q_row, k_row, v_row}, dtype)) return QA_EINVAL;
  a.q = q;
  a.k = k;
  a.v = v;
  a.dq = out;
  a.dqt = a.ot;
  a.lse = lse;
  a.rest = rest;
  return (int)launch(FORWARD, dtype, a, key_tiles_of(tokens, sequences), longest, tiles, tile_count, tile_rows, (hipStream_t)stream);
}

int qutai_amd_attention_packed_bwd(const void* grad, const void* q, const void* k, const void* v, const void* out,
                                   const void* rest, const float* lse, void* dq, void* dk, void* dv, float* delta,
                                   void* workspace, size_t workspace_bytes, const int64_t* query_tiles, int64_t query_count,
                                   int64_t query_rows, const int64_t* key_tiles, int64_t key_count, int64_t key_rows,
                                   int64_t tokens, int64_t sequences, int64_t longest, int64_t heads, int64_t kv_heads,
                                   int64_t dim, int64_t q_row, int64_t k_row, int64_t v_row, int64_t dq_row, int64_t dk_row,
                                   int64_t dv_row, int dtype, double scale, int causal, void* stream) {
  AttnPackedArgs a = {};
  const int status = set_packed(a, tokens, sequences, longest, heads, kv_heads, dim, q_row, k_row, v_row, dtype, scale, causal,
                                {{QUERIES, query_rows}, {KEYS, key_rows}});
  if (status != QA_OK) return status;
  if (dq_row < heads * dim || dk_row < kv_heads * dim || dv_row < kv_heads * dim) return QA_EINVAL;
  if (std::max({dq_row, dk_row, dv_row}) > 1 << 22) return QA_EINVAL;
  if (!grid_fits(query_count, groups_of(QUERIES, dtype, heads, kv_heads, dim, query_rows)) ||
      !grid_fits(key_count, kv_heads, heads_apart(dtype, tokens, sequences, heads, kv_heads, dim, key_rows)))
    return QA_EINVAL;
  if (!query_count && !key_count) return QA_OK;
  if (!grad || !q || !k || !v || !out || !dq || !dk || !dv || !lse || !delta || !query_tiles || !key_tiles)
    return QA_EINVAL;
  if ((query_rows != GEN_WAVES || key_rows != GEN_WAVES) &&
      !whole({grad, q, k, v, out, rest ? rest : out, dq, dk, dv}, {q_row, k_row, v_row, dq_row, dk_row, dv_row}, dtype))
    return QA_EINVAL;
  a.g = grad;
  a.q = q;
  a.k = k;
  a.v = v;
  a.o = out;
  a.rest = query_rows == GEN_WAVES || !packed_fits(dtype, dim) ? nullptr : const_cast<void*>(rest);
  a.lse = const_cast<float*>(lse);
  a.delta = delta;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.dqt = dq_row;
  a.dkt = dk_row;
  a.dvt = dv_row;
  const int64_t group = heads / kv_heads;
  const size_t need = qutai_amd_attention_packed_workspace(tokens, sequences, heads, kv_heads, dim, dtype, key_rows);
  if (need && workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0) {
    a.split = 1;
    a.part_stride = tokens * kv_heads * dim;
    a.part_k = (float*)workspace;
    a.part_v = a.part_k + group * a.part_stride;
  }
  // the query pass writes delta, which the key pass reads
  hipError_t e = launch(QUERIES, dtype, a, key_tiles_of(tokens, sequences), longest, query_tiles, query_count, query_rows,
                        (hipStream_t)stream);
  if (e != hipSuccess) return (int)e;
  e = launch(KEYS, dtype, a, key_tiles_of(tokens, sequences), longest, key_tiles, key_count, key_rows, (hipStream_t)stream);
  if (e != hipSuccess || !a.split || !key_count) return (int)e;
  const dim3 grid((unsigned)((a.part_stride / 4 + 255) / 256));
  if (dtype == BF16) hipLaunchKernelGGL(packed_dkv_sum<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, a, tokens, (int)group);
  else hipLaunchKernelGGL(packed_dkv_sum<float>, grid, dim3(256), 0, (hipStream_t)stream, a, tokens, (int)group);
  return (int)hipGetLastError();
}

}  // extern "C"
