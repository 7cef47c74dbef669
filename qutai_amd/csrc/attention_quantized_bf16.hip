// The kernels of attention_quantized.h for bf16 queries and outputs.
#include "attention_quantized.h"

int qa::attend_bf16(const void* args, const void* plan, int bits, hipStream_t stream) {
  return attend_type<bf16_t>(*(const AttendArgs*)args, *(const AttendPlan*)plan, bits, stream);
}
