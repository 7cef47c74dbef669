// A key and value cache quantised as it is written, and read back: C ABI
// `qutai_amd_cache_quantize`, `qutai_amd_cache_dequantize` (the codes and their
// layout: cache_codes.h).
#include "cache_codes.h"
#include "qutai_amd.h"

#include <initializer_list>

using namespace qa;

namespace {

constexpr int THREADS = 256;

struct WriteArgs {
  const void* x[2];  // keys, values
  uint8_t* codes[2];
  bf16_t* scales[2];
  int64_t row[2];  // elements from position to position
  const int64_t* starts;
  const int64_t* counts;
  int64_t start, batch, fresh, heads, capacity, rows;  // rows: batch x fresh x heads
  int dim, pitch;
};

template <class T> __device__ __forceinline__ float get(const T* p, int64_t i);
template <> __device__ __forceinline__ float get<float>(const float* p, int64_t i) { return p[i]; }
template <> __device__ __forceinline__ float get<bf16_t>(const bf16_t* p, int64_t i) { return bf16_to_f32(p[i]); }

// LANES lanes to a row, four channels each (a power of two of lanes; those past
// the pitch idle).
template <class T, int BITS, int LANES>
__global__ void __launch_bounds__(THREADS) cache_write(WriteArgs a) {
  const int part = threadIdx.x % LANES, d = 4 * part;
  const int64_t item = (int64_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
  const int side = blockIdx.y;
  const int64_t row = item < a.rows ? item : a.rows - 1;  // every lane takes part in the maxima
  const int64_t h = row % a.heads, at = row / a.heads, t = at % a.fresh, b = at / a.fresh;
  const int64_t position = a.start + (a.starts ? a.starts[b] : 0) + t;
  const bool there = item < a.rows && position >= 0 && position < a.capacity && (!a.counts || t < a.counts[b]);
  const T* x = (const T*)a.x[side] + at * a.row[side] + h * a.dim;
  float v[4], amax = 0.f;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    v[e] = d + e < a.dim ? get(x, d + e) : 0.f;
    const float m = fabsf(v[e]);
    amax = m <= amax || amax != amax ? amax : m;  // a NaN stays
  }
  constexpr int SPAN = BITS == 8 ? LANES : 8;
#pragma unroll
  for (int o = 1; o < SPAN; o <<= 1) {
    const float m = __shfl_xor(amax, o);
    amax = m <= amax || amax != amax ? amax : m;
  }
  const float most = BITS == 8 ? 127.f : 7.f;
  const uint32_t bits = scale_bits(amax, most);
  const float s = __uint_as_float(bits << 16), inverse = 1.f / s;
  int q[4];
#pragma unroll
  for (int e = 0; e < 4; e++) q[e] = bits == 0x7fc0u ? 0 : code_of(v[e], s, inverse);
  if (!there || d >= a.pitch) return;
  const int64_t slot = (b * a.heads + h) * a.capacity + position;
  if constexpr (BITS == 8) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) w |= (uint32_t)(q[e] & 255) << (8 * e);
    *(uint32_t*)(a.codes[side] + slot * a.pitch + d) = w;
    if (part == 0) a.scales[side][slot] = (bf16_t)bits;
  } else {
    uint8_t* out = a.codes[side] + slot * (a.pitch / 2);
    const int groups = a.pitch / 32;
    if (side == 0) {  // a dword of eight channels: nibbles 0 4 1 5 here, 2 6 3 7 in the next lane
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) w |= (uint32_t)(q[e] & 15) << (4 * ((e >> 1) + 4 * (e & 1) + 2 * (part & 1)));
      w |= __shfl_xor(w, 1);
      if ((part & 1) == 0) *(uint32_t*)(out + ((d >> 3) & 3) * (a.pitch >> 3) + 4 * (d >> 5)) = w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        int shift;
        out[value_nibble(d + e, a.pitch, shift)] = (uint8_t)((q[e] & 15) | (q[e + 1] & 15) << 4);
      }
    }
    if ((part & 7) == 0) a.scales[side][slot * groups + (part >> 3)] = (bf16_t)bits;
  }
}

struct ReadArgs {
  const uint8_t* codes;
  const bf16_t* scales;
  void* out;
  const int64_t* lengths;
  int64_t shift, heads, capacity, length, rows;  // rows: batch x heads x length
  int dim, pitch, keys;
};

template <class T, int BITS>
__global__ void __launch_bounds__(THREADS) cache_read(ReadArgs a) {
  const int parts = (a.dim + 3) / 4;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < a.rows * parts; i += (int64_t)gridDim.x * THREADS) {
    const int64_t row = i / parts, t = row % a.length, bh = row / a.length;
    const int d = 4 * (int)(i % parts);
    const int64_t slot = bh * a.capacity + t;
    const bool there = t < a.shift + (a.lengths ? a.lengths[bh / a.heads] : 0);
    T* out = (T*)a.out + row * a.dim;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (d + e >= a.dim) break;
      float v = 0.f;
      if (there) {
        if constexpr (BITS == 8) {
          v = (float)(int8_t)a.codes[slot * a.pitch + d + e] * bf16_to_f32(a.scales[slot]);
        } else {
          int shift;
          const int at = a.keys ? key_nibble(d + e, a.pitch, shift) : value_nibble(d + e, a.pitch, shift);
          v = (float)nibble_value(a.codes[slot * (a.pitch / 2) + at], shift) *
              bf16_to_f32(a.scales[slot * (a.pitch / 32) + ((d + e) >> 5)]);
        }
      }
      if constexpr (sizeof(T) == 2) out[d + e] = f32_to_bf16(v);
      else out[d + e] = v;
    }
  }
}

template <class T, int BITS>
void launch_write(const WriteArgs& a, hipStream_t stream) {
  const int lanes = a.pitch / 4;
  auto grid = [&](int per) { return dim3((unsigned)((a.rows + THREADS / per - 1) / (THREADS / per)), 2); };
  if (lanes <= 8) hipLaunchKernelGGL((cache_write<T, BITS, 8>), grid(8), dim3(THREADS), 0, stream, a);
  else if (lanes <= 16) hipLaunchKernelGGL((cache_write<T, BITS, 16>), grid(16), dim3(THREADS), 0, stream, a);
  else if (lanes <= 32) hipLaunchKernelGGL((cache_write<T, BITS, 32>), grid(32), dim3(THREADS), 0, stream, a);
  else hipLaunchKernelGGL((cache_write<T, BITS, 64>), grid(64), dim3(THREADS), 0, stream, a);
}

bool sizes_ok(int64_t batch, int64_t heads, int64_t dim, int64_t capacity, int bits, int dtype) {
  return batch >= 0 && heads > 0 && heads <= 65536 && dim > 0 && dim <= 256 && capacity > 0 && capacity <= (1ll << 30) &&
         batch <= (1ll << 24) && (bits == 8 || bits == 4) && (dtype == BF16 || dtype == F32);
}

}  // namespace

extern "C" int64_t qutai_amd_cache_pitch(int64_t dim) { return dim > 0 && dim <= 256 ? cache_pitch(dim) : 0; }

extern "C" int qutai_amd_cache_quantize(const void* keys, const void* values, void* key_codes, void* key_scales,
                                        void* value_codes, void* value_scales, const int64_t* starts,
                                        const int64_t* counts, int64_t start, int64_t batch, int64_t fresh,
                                        int64_t kv_heads, int64_t dim, int64_t capacity, int64_t key_row,
                                        int64_t value_row, int bits, int dtype, void* stream_) {
  if (!sizes_ok(batch, kv_heads, dim, capacity, bits, dtype) || fresh < 0 || fresh > (1ll << 31)) return QA_EINVAL;
  if (key_row < kv_heads * dim || value_row < kv_heads * dim || key_row > (1ll << 40) || value_row > (1ll << 40))
    return QA_EINVAL;
  if (start < -(1ll << 40) || start > (1ll << 40)) return QA_EINVAL;
  if (batch == 0 || fresh == 0) return QA_OK;
  const int64_t most = 1ll << 28;  // rows: below 2^32 threads in a launch, 64 lanes to a row at most, and keys and values
  if (fresh > most / batch || batch * fresh > most / kv_heads / 8 || (int64_t)capacity * kv_heads > (1ll << 44) / batch)
    return QA_EINVAL;
  for (const int64_t row : {key_row, value_row})
    if (batch * fresh > (1ll << 60) / row) return QA_EINVAL;
  for (const void* p : {keys, values, (const void*)key_codes, (const void*)key_scales, (const void*)value_codes,
                        (const void*)value_scales})
    if (!p) return QA_EINVAL;
  if ((uintptr_t)key_codes % 16 || (uintptr_t)value_codes % 16) return QA_EINVAL;
  const WriteArgs a = {{keys, values}, {(uint8_t*)key_codes, (uint8_t*)value_codes},
                       {(bf16_t*)key_scales, (bf16_t*)value_scales}, {key_row, value_row}, starts, counts, start, batch,
                       fresh, kv_heads, capacity, batch * fresh * kv_heads, (int)dim, (int)cache_pitch(dim)};
  hipStream_t stream = (hipStream_t)stream_;
  if (dtype == BF16) {
    if (bits == 8) launch_write<bf16_t, 8>(a, stream);
    else launch_write<bf16_t, 4>(a, stream);
  } else {
    if (bits == 8) launch_write<float, 8>(a, stream);
    else launch_write<float, 4>(a, stream);
  }
  return (int)hipGetLastError();
}

extern "C" int qutai_amd_cache_dequantize(const void* codes, const void* scales, void* out, const int64_t* lengths,
                                          int64_t shift, int64_t batch, int64_t kv_heads, int64_t dim, int64_t capacity,
                                          int64_t length, int bits, int keys, int dtype, void* stream_) {
  if (!sizes_ok(batch, kv_heads, dim, capacity, bits, dtype) || length < 0 || length > capacity) return QA_EINVAL;
  if (shift < -(1ll << 40) || shift > (1ll << 40)) return QA_EINVAL;
  if (batch == 0 || length == 0) return QA_OK;
  if ((int64_t)capacity * kv_heads > (1ll << 44) / batch || !codes || !scales || !out || (uintptr_t)codes % 16)
    return QA_EINVAL;
  const ReadArgs a = {(const uint8_t*)codes, (const bf16_t*)scales, out, lengths, shift, kv_heads, capacity, length,
                      batch * kv_heads * length, (int)dim, (int)cache_pitch(dim), keys ? 1 : 0};
  const int64_t blocks = (a.rows * ((dim + 3) / 4) + THREADS - 1) / THREADS;
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20));
  hipStream_t stream = (hipStream_t)stream_;
  if (dtype == BF16) {
    if (bits == 8) hipLaunchKernelGGL((cache_read<bf16_t, 8>), grid, dim3(THREADS), 0, stream, a);
    else hipLaunchKernelGGL((cache_read<bf16_t, 4>), grid, dim3(THREADS), 0, stream, a);
  } else {
    if (bits == 8) hipLaunchKernelGGL((cache_read<float, 8>), grid, dim3(THREADS), 0, stream, a);
    else hipLaunchKernelGGL((cache_read<float, 4>), grid, dim3(THREADS), 0, stream, a);
  }
  return (int)hipGetLastError();
}
