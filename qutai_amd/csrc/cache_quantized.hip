// A key and value cache quantised as it is written, and read back: C ABI
// `qutai_amd_cache_quantize`, `qutai_amd_cache_dequantize` (the codes and their
// layout: cache_codes.h).  Bound by HBM: 4 x 4000 positions of 8 heads of 128, keys
// and values, bf16 to 8 bits: 24 us to write (98 MB, 4.1 TB/s; four channels per
// lane and 64-bit row arithmetic 57), 16 us to read back (6.2 TB/s; 44 in two
// launches of four channels per lane).
#include "cache_codes.h"
#include "qutai_amd.h"

#include <initializer_list>
#include <type_traits>

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
  int64_t start, capacity;
  uint32_t fresh, heads, rows;  // rows: batch x fresh x heads, at most 2^25
  int dim, pitch, vector;
};

template <class T> __device__ __forceinline__ float get(const T* p, int64_t i);
template <> __device__ __forceinline__ float get<float>(const float* p, int64_t i) { return p[i]; }
template <> __device__ __forceinline__ float get<bf16_t>(const bf16_t* p, int64_t i) { return bf16_to_f32(p[i]); }

// eight channels of a row from channel d on, zeros behind its last
template <class T>
__device__ __forceinline__ void load8(const T* x, int d, int dim, bool vector, float (&v)[8]) {
  if (vector && d + 8 <= dim) {
    if constexpr (sizeof(T) == 2) {
      const u32x4 w = global_load<u32x4>(x + d);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    } else {
      const u32x4 a = global_load<u32x4>(x + d), b = global_load<u32x4>(x + d + 4);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = __uint_as_float(e < 4 ? a[e] : b[e - 4]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = d + e < dim ? get(x, d + e) : 0.f;
  }
}

// Eight channels per lane, LANES lanes to a row (a power of two; those past the
// pitch idle), U rows per lane in flight.  Bound by HBM: a row is read once, 16
// bytes per lane, and its codes written once.
template <class T, int BITS, int LANES>
__global__ void __launch_bounds__(THREADS) cache_write(WriteArgs a) {
  constexpr int U = sizeof(T) == 2 ? 4 : 2;
  const int part = threadIdx.x % LANES, d = 8 * part, side = blockIdx.y;
  const bool inside = d < a.pitch;
  float v[U][8];
  int64_t slot[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t item = (blockIdx.x * U + u) * (THREADS / LANES) + threadIdx.x / LANES;
    const uint32_t row = item < a.rows ? item : a.rows - 1;  // every lane takes part in the maxima
    const uint32_t at = row / a.heads, h = row - at * a.heads, b = at / a.fresh, t = at - b * a.fresh;
    const int64_t position = a.start + (a.starts ? a.starts[b] : 0) + t;
    const bool there = item < a.rows && position >= 0 && position < a.capacity && (!a.counts || (int64_t)t < a.counts[b]);
    slot[u] = there && inside ? (int64_t)(b * a.heads + h) * a.capacity + position : -1;
    load8((const T*)a.x[side] + (int64_t)at * a.row[side] + h * a.dim, d, a.dim, a.vector, v[u]);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float m = fabsf(v[u][e]);
      amax = m <= amax || amax != amax ? amax : m;  // a NaN stays
    }
    constexpr int SPAN = BITS == 8 ? LANES : 4;
#pragma unroll
    for (int o = 1; o < SPAN; o <<= 1) {
      const float m = __shfl_xor(amax, o);
      amax = m <= amax || amax != amax ? amax : m;
    }
    const uint32_t bits = scale_bits(amax, BITS == 8 ? 127.f : 7.f);
    const float s = __uint_as_float(bits << 16), inverse = 1.f / s;
    uint32_t q[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float c = sizeof(T) == 2 ? code_of_bf16(v[u][e], inverse) : code_of(v[u][e], s, inverse);
      q[e] = low_byte(bits == 0x7fc0u ? 0.f : c);
    }
    if (slot[u] < 0) continue;
    if constexpr (BITS == 8) {
      u32x2 w;
#pragma unroll
      for (int i = 0; i < 2; i++)
        w[i] = (q[4 * i] & 255) | (q[4 * i + 1] & 255) << 8 | (q[4 * i + 2] & 255) << 16 | q[4 * i + 3] << 24;
      global_store(a.codes[side] + slot[u] * a.pitch + d, w);
      if (part == 0) a.scales[side][slot[u]] = (bf16_t)bits;
    } else {
      uint8_t* out = a.codes[side] + slot[u] * (a.pitch / 2);
      if (side == 0) {  // a dword: nibble n is channel 2 (n % 4) + n / 4 of the eight
        uint32_t w = 0;
#pragma unroll
        for (int n = 0; n < 8; n++) w |= (q[2 * (n & 3) + (n >> 2)] & 15) << (4 * n);
        *(uint32_t*)(out + (part & 3) * (a.pitch >> 3) + 4 * (part >> 2)) = w ^ 0x88888888u;
      } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          out[(4 * (part & 3) + e / 2) * (a.pitch >> 5) + (part >> 2)] = (uint8_t)(((q[e] & 15) | (q[e + 1] & 15) << 4) ^ 0x88);
      }
      if ((part & 3) == 0) a.scales[side][slot[u] * (a.pitch / 32) + (part >> 2)] = (bf16_t)bits;
    }
  }
}

struct ReadArgs {
  const uint8_t* codes[2];
  const bf16_t* scales[2];
  void* out[2];
  const int64_t* lengths;
  int64_t shift, capacity;
  uint32_t heads, length, rows;  // rows: batch x heads x length
  int dim, pitch, vector;
};

// The reverse, laid out the same way: rows are [batch][heads][length].
template <class T, int BITS, int LANES>
__global__ void __launch_bounds__(THREADS) cache_read(ReadArgs a) {
  constexpr int U = 4;
  const int part = threadIdx.x % LANES, d = 8 * part, side = blockIdx.y;
  if (d >= a.dim) return;
  u32x2 code[U];
  float scale[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t row = (blockIdx.x * U + u) * (THREADS / LANES) + threadIdx.x / LANES;
    code[u] = u32x2{0u, 0u}, scale[u] = 0.f;
    if (row >= a.rows) continue;
    const uint32_t bh = row / a.length, t = row - bh * a.length, b = bh / a.heads;
    if ((int64_t)t >= a.shift + (a.lengths ? a.lengths[b] : 0)) continue;
    const int64_t slot = (int64_t)bh * a.capacity + t;
    if constexpr (BITS == 8) {
      code[u] = global_load<u32x2>(a.codes[side] + slot * a.pitch + d);
      scale[u] = bf16_to_f32(a.scales[side][slot]);
    } else {
      const uint8_t* p = a.codes[side] + slot * (a.pitch / 2);
      if (side == 0) {
        code[u][0] = global_load<uint32_t>(p + (part & 3) * (a.pitch >> 3) + 4 * (part >> 2));
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) code[u][0] |= (uint32_t)p[(4 * (part & 3) + e) * (a.pitch >> 5) + (part >> 2)] << (8 * e);
      }
      scale[u] = bf16_to_f32(a.scales[side][slot * (a.pitch / 32) + (part >> 2)]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t row = (blockIdx.x * U + u) * (THREADS / LANES) + threadIdx.x / LANES;
    if (row >= a.rows) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      int c;
      if constexpr (BITS == 8) c = (int8_t)(code[u][e >> 2] >> (8 * (e & 3)));
      else c = (int)(code[u][0] >> (4 * (side == 0 ? (e >> 1) + 4 * (e & 1) : e)) & 15) - 8;
      v[e] = (float)c * scale[u];
    }
    T* out = (T*)a.out[side] + (int64_t)row * a.dim;
    if (a.vector && d + 8 <= a.dim) {
      if constexpr (sizeof(T) == 2) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
        global_store(out + d, w);
      } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const f32x4 w = {v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
          global_store(out + d + 4 * i, w);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if (d + e >= a.dim) break;
        if constexpr (sizeof(T) == 2) out[d + e] = f32_to_bf16(v[e]);
        else out[d + e] = v[e];
      }
    }
  }
}

// launch(LANES) with the lanes of a row: eight channels each, a power of two
template <class F>
void by_lanes(int pitch, F launch) {
  if (pitch <= 32) launch(std::integral_constant<int, 4>());
  else if (pitch <= 64) launch(std::integral_constant<int, 8>());
  else if (pitch <= 128) launch(std::integral_constant<int, 16>());
  else launch(std::integral_constant<int, 32>());
}

template <class T, int BITS>
void launch_write(const WriteArgs& a, hipStream_t stream) {
  by_lanes(a.pitch, [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value, ROWS = THREADS / LANES * (sizeof(T) == 2 ? 4 : 2);
    hipLaunchKernelGGL((cache_write<T, BITS, LANES>), dim3((a.rows + ROWS - 1) / ROWS, 2), dim3(THREADS), 0, stream, a);
  });
}

template <class T, int BITS>
void launch_read(const ReadArgs& a, hipStream_t stream) {
  by_lanes(a.pitch, [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value, ROWS = THREADS / LANES * 4;
    hipLaunchKernelGGL((cache_read<T, BITS, LANES>), dim3((a.rows + ROWS - 1) / ROWS, 2), dim3(THREADS), 0, stream, a);
  });
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
  const int64_t most = 1ll << 25;  // rows: 32 lanes each at most, a lane has two or four: 2^30 threads for keys and values
  if (fresh > most / batch || batch * fresh > most / kv_heads || (int64_t)capacity * kv_heads > (1ll << 44) / batch)
    return QA_EINVAL;
  for (const int64_t row : {key_row, value_row})
    if (batch * fresh > (1ll << 60) / row) return QA_EINVAL;
  for (const void* p : {keys, values, (const void*)key_codes, (const void*)key_scales, (const void*)value_codes,
                        (const void*)value_scales})
    if (!p) return QA_EINVAL;
  if ((uintptr_t)key_codes % 16 || (uintptr_t)value_codes % 16) return QA_EINVAL;
  const int64_t es = dtype == BF16 ? 2 : 4;
  const bool vector = dim % 8 == 0 && key_row * es % 16 == 0 && value_row * es % 16 == 0 && (uintptr_t)keys % 16 == 0 &&
                      (uintptr_t)values % 16 == 0;
  const WriteArgs a = {{keys, values}, {(uint8_t*)key_codes, (uint8_t*)value_codes},
                       {(bf16_t*)key_scales, (bf16_t*)value_scales}, {key_row, value_row}, starts, counts, start, capacity,
                       (uint32_t)fresh, (uint32_t)kv_heads, (uint32_t)(batch * fresh * kv_heads), (int)dim,
                       (int)cache_pitch(dim), vector};
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

extern "C" int qutai_amd_cache_dequantize(const void* key_codes, const void* key_scales, const void* value_codes,
                                          const void* value_scales, void* keys, void* values, const int64_t* lengths,
                                          int64_t shift, int64_t batch, int64_t kv_heads, int64_t dim, int64_t capacity,
                                          int64_t length, int bits, int dtype, void* stream_) {
  if (!sizes_ok(batch, kv_heads, dim, capacity, bits, dtype) || length < 0 || length > capacity) return QA_EINVAL;
  if (shift < -(1ll << 40) || shift > (1ll << 40)) return QA_EINVAL;
  if (batch == 0 || length == 0) return QA_OK;
  // rows: below 2^32 threads in a launch, 32 lanes to a row at most, four rows to a lane, two sides
  if (length > (1ll << 28) / batch || batch * length > (1ll << 28) / kv_heads) return QA_EINVAL;
  if ((int64_t)capacity * kv_heads > (1ll << 44) / batch) return QA_EINVAL;
  for (const void* p : {key_codes, key_scales, value_codes, value_scales, (const void*)keys, (const void*)values})
    if (!p) return QA_EINVAL;
  if ((uintptr_t)key_codes % 16 || (uintptr_t)value_codes % 16) return QA_EINVAL;
  const bool vector = dim % 8 == 0 && (uintptr_t)keys % 16 == 0 && (uintptr_t)values % 16 == 0;
  const ReadArgs a = {{(const uint8_t*)key_codes, (const uint8_t*)value_codes},
                      {(const bf16_t*)key_scales, (const bf16_t*)value_scales}, {keys, values}, lengths, shift, capacity,
                      (uint32_t)kv_heads, (uint32_t)length, (uint32_t)(batch * kv_heads * length), (int)dim,
                      (int)cache_pitch(dim), vector};
  hipStream_t stream = (hipStream_t)stream_;
  if (dtype == BF16) {
    if (bits == 8) launch_read<bf16_t, 8>(a, stream);
    else launch_read<bf16_t, 4>(a, stream);
  } else {
    if (bits == 8) launch_read<float, 8>(a, stream);
    else launch_read<float, 4>(a, stream);
  }
  return (int)hipGetLastError();
}
