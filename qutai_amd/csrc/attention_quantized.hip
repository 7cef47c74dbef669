// Attention of new positions over a quantised key and value cache: C ABI
// `qutai_amd_attention_quantized` and its plan (the kernels:
// attention_quantized.h).
#include "attention_quantized.h"

#include <initializer_list>

namespace {

// Workgroups wanted in a launch of 256 CUs.  Where a tile has few rows, and the keys
// are what is read: two for each, which run together (16 sequences of up to 7000
// keys, 4 bits, 128 channels: 31 us, 35 with four, 41 with six); four, which even
// out sequences of different lengths, where a range keeps LONG_RANGE keys all the
// same (32 of up to 14000, 8 bits: 120 us, 132 with two, 128 with six).  Where it
// has many rows, whose sums a split one writes and reads again: one (512 new
// positions over 3500: 63 us, 79 with two, 96 with four).
// Few rows are those that share a tile (bf16 8 and fewer, fp32 4).  From there to
// some 32 rows the keys of a long cache bound a call as before, and it would gain
// from the ranges of few rows, which it does not get: 32 sequences of up to 14000, 8
// bits, bf16, 8 kv heads of 128: 129 us with 8 rows, 200 with 9 to 17, 209 with 32 (150
// to 157, and 167); 16 of up to 8000, 4 bits: 43 with 8, 82 with 9 (71); fp32, 16 of
// up to 7000, 8 bits: 41 with 4, 64 to 69 with 5 to 17 (62 to 68), 73 with 32 (76).
constexpr int64_t FEW_ROWS = 512, MANY_ROWS = 256, LONG_RANGE = 2048;

AttendPlan plan_of(int64_t batch, int64_t fresh, int64_t heads, int64_t kv_heads, int64_t dim, int64_t longest, int bits,
                   int dtype) {
  AttendPlan p;
  const int item = dtype == BF16 ? 2 : 4;
  const int64_t rows = fresh * (heads / kv_heads);
  p.pitch = (int)cache_pitch(dim);
  p.spread = rows <= 4 ? 4 : dtype == BF16 && rows <= 8 ? 2 : 1;
  p.tile = p.spread > 1 || one_tile(item, bits, p.pitch) ? 1 : dtype == F32 || p.pitch > 128 || rows <= 32 ? 2 : 4;
  p.rows = 16 / p.spread * p.tile;
  p.tiles = (rows + p.rows - 1) / p.rows;
  const int64_t units = batch * kv_heads * p.tiles;
  const int64_t step = WAVES * BLOCK * (p.spread == 4 ? blocks_of(item, bits, p.pitch) : 1);
  const int64_t most = (longest + step - 1) / step;
  p.splits = ((p.spread > 1 ? FEW_ROWS : MANY_ROWS) + units - 1) / units;
  if (p.spread > 1 && longest / ((2 * FEW_ROWS + units - 1) / units) >= LONG_RANGE) p.splits = (2 * FEW_ROWS + units - 1) / units;
  if (p.splits > most) p.splits = most;
  if (p.splits > 256) p.splits = 256;
  if (p.splits < 1) p.splits = 1;
  return p;
}

int64_t slots_of(const AttendPlan& p, int64_t units) { return units * p.tiles * p.splits * p.rows; }

bool sizes_ok(int64_t batch, int64_t fresh, int64_t heads, int64_t kv_heads, int64_t dim, int64_t longest, int dtype) {
  return batch >= 0 && fresh >= 0 && heads > 0 && heads <= 65536 && kv_heads > 0 && heads % kv_heads == 0 && dim > 0 &&
         dim <= 256 && longest >= 0 && longest <= (1ll << 30) && (dtype == BF16 || dtype == F32) && batch <= (1ll << 24) &&
         fresh <= (1ll << 24) && batch * fresh <= (1ll << 25) / heads && batch * kv_heads <= (1ll << 22);
}

}  // namespace

extern "C" size_t qutai_amd_attention_quantized_workspace_size(int64_t batch, int64_t fresh, int64_t heads,
                                                               int64_t kv_heads, int64_t dim, int64_t longest, int dtype) {
  if (!sizes_ok(batch, fresh, heads, kv_heads, dim, longest, dtype) || batch == 0 || fresh == 0) return 0;
  size_t need = 0;
  for (const int bits : {8, 4}) {
    const AttendPlan p = plan_of(batch, fresh, heads, kv_heads, dim, longest, bits, dtype);
    const size_t own = p.splits > 1 ? (size_t)slots_of(p, batch * kv_heads) * (p.pitch + 2) * sizeof(float) : 0;
    need = own > need ? own : need;
  }
  return need;
}

extern "C" int qutai_amd_attention_quantized(const void* q, const void* key_codes, const void* key_scales,
                                             const void* value_codes, const void* value_scales, void* out,
                                             const int64_t* starts, const int64_t* counts, int64_t start, int64_t batch,
                                             int64_t fresh, int64_t heads, int64_t kv_heads, int64_t dim,
                                             int64_t capacity, int64_t longest, int bits, int dtype, double scale,
                                             void* workspace, size_t workspace_bytes, void* stream_) {
  if (!sizes_ok(batch, fresh, heads, kv_heads, dim, longest, dtype)) return QA_EINVAL;
  if (capacity <= 0 || capacity % 32 || capacity > (1ll << 30) || longest > capacity) return QA_EINVAL;
  if ((bits != 8 && bits != 4) || !(scale >= 1e-30) || scale > 1e30) return QA_EINVAL;
  if (start < -(1ll << 40) || start > (1ll << 40)) return QA_EINVAL;
  if (batch == 0 || fresh == 0) return QA_OK;
  if (capacity * kv_heads > (1ll << 44) / batch) return QA_EINVAL;
  if (!q || !key_codes || !key_scales || !value_codes || !value_scales || !out) return QA_EINVAL;
  if ((uintptr_t)key_codes % 16 || (uintptr_t)value_codes % 16 || (uintptr_t)key_scales % 4 || (uintptr_t)value_scales % 4)
    return QA_EINVAL;
  const AttendPlan p = plan_of(batch, fresh, heads, kv_heads, dim, longest, bits, dtype);
  const int64_t units = batch * kv_heads;
  if (units * p.tiles * p.splits >= (1ll << 24)) return QA_EINVAL;  // workgroups of 256 threads, below 2^32
  const int64_t slots = slots_of(p, units);
  if (p.splits > 1 && (!workspace || (uintptr_t)workspace % 4 ||
                       workspace_bytes < (size_t)slots * (p.pitch + 2) * sizeof(float)))
    return QA_EWORKSPACE;
  float* part = (float*)workspace;
  const AttendArgs a = {q, {(const uint8_t*)key_codes, (const uint8_t*)value_codes},
                        {(const bf16_t*)key_scales, (const bf16_t*)value_scales}, out, starts, counts, part,
                        part ? part + slots * p.pitch : nullptr, start, fresh, heads, kv_heads, capacity, units,
                        (int)(heads / kv_heads), (int)dim, dtype == BF16 && dim % 8 == 0 && (uintptr_t)q % 16 == 0,
                        (int)p.tiles, (int)p.splits, (float)(scale * 1.4426950408889634)};
  hipStream_t stream = (hipStream_t)stream_;
  return dtype == BF16 ? attend_bf16(&a, &p, bits, stream) : attend_fp32(&a, &p, bits, stream);
}
