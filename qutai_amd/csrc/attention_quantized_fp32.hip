// The kernels of attention_quantized.h for fp32 queries and outputs.
#include "attention_quantized.h"

int qa::attend_fp32(const void* args, const void* plan, int bits, hipStream_t stream) {
  return attend_type<float>(*(const AttendArgs*)args, *(const AttendPlan*)plan, bits, stream);
}
