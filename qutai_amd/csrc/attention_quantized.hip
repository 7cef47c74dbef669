// Attention of new positions over a quantised key and value cache: C ABI
// `qutai_amd_attention_quantized` (the codes and their layout: cache_codes.h).
//
// Query t of sequence b stands at position p = start + starts[b] + t and sees
// the keys 0 .. p:  o = sum_j softmax_j(scale q . k_j) v_j, with k_j and v_j the
// values that the codes stand for.
#include "cache_codes.h"
#include "qutai_amd.h"

using namespace qa;

namespace {

struct AttendArgs {
  const void* q;
  const uint8_t* codes[2];
  const bf16_t* scales[2];
  void* out;
  const int64_t* starts;
  const int64_t* counts;
  int64_t start, batch, fresh, heads, kv_heads, capacity;
  int dim, pitch;
  float scale;
};

template <class T> __device__ __forceinline__ float get(const T* p, int64_t i);
template <> __device__ __forceinline__ float get<float>(const float* p, int64_t i) { return p[i]; }
template <> __device__ __forceinline__ float get<bf16_t>(const bf16_t* p, int64_t i) { return bf16_to_f32(p[i]); }

template <int BITS>
__device__ __forceinline__ float held(const AttendArgs& a, int side, int64_t slot, int d) {
  if constexpr (BITS == 8) {
    return (float)(int8_t)a.codes[side][slot * a.pitch + d] * bf16_to_f32(a.scales[side][slot]);
  } else {
    int shift;
    const int at = side == 0 ? key_nibble(d, a.pitch, shift) : value_nibble(d, a.pitch, shift);
    return (float)nibble_value(a.codes[side][slot * (a.pitch / 2) + at], shift) *
           bf16_to_f32(a.scales[side][slot * (a.pitch / 32) + (d >> 5)]);
  }
}

// A wave per query and head: 64 keys at a time, a key per lane for the scores,
// channels over the lanes for the values.
template <class T, int BITS>
__global__ void __launch_bounds__(64) attend_rows(AttendArgs a) {
  __shared__ float q[256];
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x, h = row % a.heads, at = row / a.heads, t = at % a.fresh, b = at / a.fresh;
  T* out = (T*)a.out + row * a.dim;
  const int64_t position = a.start + (a.starts ? a.starts[b] : 0) + t;
  int64_t visible = position + 1 < a.capacity ? position + 1 : a.capacity;
  if (a.counts && t >= a.counts[b]) visible = 0;
  for (int d = lane; d < a.dim; d += 64) q[d] = get((const T*)a.q, row * a.dim + d);
  __syncthreads();
  const int64_t first = (b * a.kv_heads + h / (a.heads / a.kv_heads)) * a.capacity;
  float top = -INFINITY, total = 0.f, acc[4] = {};
  for (int64_t s0 = 0; s0 < visible; s0 += 64) {
    const int64_t s = s0 + lane;
    float score = -INFINITY;
    if (s < visible) {
      score = 0.f;
      for (int d = 0; d < a.dim; d++) score = fmaf(q[d], held<BITS>(a, 0, first + s, d), score);
      score *= a.scale;
    }
    float m = score;
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    m = fmaxf(m, top);
    const float fade = __expf(top - m), p = __expf(score - m);
    top = m;
    total = total * fade + p;
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] *= fade;
    const int n = (int)(visible - s0 < 64 ? visible - s0 : 64);
    for (int j = 0; j < n; j++) {
      const float w = __shfl(p, j);
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (lane + 64 * e < a.dim) acc[e] = fmaf(w, held<BITS>(a, 1, first + s0 + j, lane + 64 * e), acc[e]);
    }
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int d = lane + 64 * e;
    if (d >= a.dim) continue;
    const float v = visible > 0 ? acc[e] / total : 0.f;
    if constexpr (sizeof(T) == 2) out[d] = f32_to_bf16(v);
    else out[d] = v;
  }
}

}  // namespace

extern "C" int qutai_amd_attention_quantized(const void* q, const void* key_codes, const void* key_scales,
                                             const void* value_codes, const void* value_scales, void* out,
                                             const int64_t* starts, const int64_t* counts, int64_t start, int64_t batch,
                                             int64_t fresh, int64_t heads, int64_t kv_heads, int64_t dim,
                                             int64_t capacity, int64_t longest, int bits, int dtype, double scale,
                                             void* workspace, size_t workspace_bytes, void* stream_) {
  (void)workspace, (void)workspace_bytes;
  if (batch < 0 || fresh < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > 65536) return QA_EINVAL;
  if (dim <= 0 || dim > 256 || capacity <= 0 || capacity > (1ll << 31) || longest < 0 || longest > capacity)
    return QA_EINVAL;
  if ((bits != 8 && bits != 4) || (dtype != BF16 && dtype != F32) || !(scale > 0.0) || scale > 1e30) return QA_EINVAL;
  if (start < -(1ll << 40) || start > (1ll << 40)) return QA_EINVAL;
  if (batch == 0 || fresh == 0) return QA_OK;
  if (batch > (1ll << 24) || fresh > (1ll << 24) || batch * fresh > (1ll << 25) / heads) return QA_EINVAL;
  if (capacity * kv_heads > (1ll << 44) / batch) return QA_EINVAL;
  if (!q || !key_codes || !key_scales || !value_codes || !value_scales || !out) return QA_EINVAL;
  if ((uintptr_t)key_codes % 16 || (uintptr_t)value_codes % 16) return QA_EINVAL;
  const AttendArgs a = {q, {(const uint8_t*)key_codes, (const uint8_t*)value_codes},
                        {(const bf16_t*)key_scales, (const bf16_t*)value_scales}, out, starts, counts, start, batch,
                        fresh, heads, kv_heads, capacity, (int)dim, (int)cache_pitch(dim), (float)scale};
  const dim3 grid((unsigned)(batch * fresh * heads));
  hipStream_t stream = (hipStream_t)stream_;
  if (dtype == BF16) {
    if (bits == 8) hipLaunchKernelGGL((attend_rows<bf16_t, 8>), grid, dim3(64), 0, stream, a);
    else hipLaunchKernelGGL((attend_rows<bf16_t, 4>), grid, dim3(64), 0, stream, a);
  } else {
    if (bits == 8) hipLaunchKernelGGL((attend_rows<float, 8>), grid, dim3(64), 0, stream, a);
    else hipLaunchKernelGGL((attend_rows<float, 4>), grid, dim3(64), 0, stream, a);
  }
  return (int)hipGetLastError();
}

extern "C" size_t qutai_amd_attention_quantized_workspace_size(int64_t batch, int64_t fresh, int64_t heads,
                                                               int64_t kv_heads, int64_t dim, int64_t longest) {
  (void)batch, (void)fresh, (void)heads, (void)kv_heads, (void)dim, (void)longest;
  return 0;
}
