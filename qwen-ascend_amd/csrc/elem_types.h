// Element types of the kernels that take bf16, fp16 and fp32 tensors.
#pragma once
#include "qmoe.h"
#include "qmoe_common.h"

struct ElemBF16 {
  using raw = uint16_t;
  QMOE_DEV static float load(raw v) { return bf16_to_f32(v); }
  QMOE_DEV static raw store(float f) { return (raw)f32_to_bf16(f); }
};
struct ElemF16 {
  using raw = uint16_t;
  QMOE_DEV static float load(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
  QMOE_DEV static raw store(float f) { return __builtin_bit_cast(raw, (_Float16)f); }
};
struct ElemF32 {
  using raw = float;
  QMOE_DEV static float load(raw v) { return v; }
  QMOE_DEV static raw store(float f) { return f; }
};

// Element i of a tensor whose type is known at run time only.
QMOE_DEV float load_typed(const void* p, long i, int type) {
  if (type == QMOE_F32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return type == QMOE_BF16 ? ElemBF16::load(v) : ElemF16::load(v);
}

static inline bool known_type(int t) { return t == QMOE_BF16 || t == QMOE_F16 || t == QMOE_F32; }
