// Element types of the kernels that take bf16, fp16 and fp32 tensors.
#pragma once
#include "qmoe.h"
#include "qmoe_common.h"

struct ElemBF16 {
  using raw = uint16_t;
  // two values as one word (hardware conversion, round to nearest even)
  QMOE_DEV static uint32_t pack(float lo, float hi) { return pk_bf16(lo, hi); }
  QMOE_DEV static float load(raw v) { return bf16_to_f32(v); }
  QMOE_DEV static raw store(float f) { return (raw)f32_to_bf16(f); }
};
struct ElemF16 {
  using raw = uint16_t;
  QMOE_DEV static uint32_t pack(float lo, float hi) { return (uint32_t)store(lo) | ((uint32_t)store(hi) << 16); }
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

// 16 bytes at any alignment of the elements: one load or store all the same (the target's
// global accesses need no alignment).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

// N consecutive elements of a type of `BYTES` each, as loaded: whole words, nothing converted
// yet, so that several can be in flight.
template <int N, int BYTES>
struct RawVec {
  static constexpr int WORDS = N * BYTES / 4;
  uint32_t w[WORDS];

  // elements [0, N) from p
  QMOE_DEV void load(const void* p) {
    if constexpr (WORDS == 2) {
      const u32x2_any v = *static_cast<const u32x2_any*>(p);
      w[0] = v[0], w[1] = v[1];
    } else {
#pragma unroll
      for (int q = 0; q < WORDS; q += 4) {
        const u32x4_any v = static_cast<const u32x4_any*>(p)[q / 4];
        w[q] = v[0], w[q + 1] = v[1], w[q + 2] = v[2], w[q + 3] = v[3];
      }
    }
  }
  QMOE_DEV void zero() {
#pragma unroll
    for (int q = 0; q < WORDS; ++q) w[q] = 0;
  }
  QMOE_DEV void store(void* p) const {
    if constexpr (WORDS == 2) {
      *static_cast<u32x2_any*>(p) = (u32x2_any){w[0], w[1]};
    } else {
#pragma unroll
      for (int q = 0; q < WORDS; q += 4) static_cast<u32x4_any*>(p)[q / 4] = (u32x4_any){w[q], w[q + 1], w[q + 2], w[q + 3]};
    }
  }
  template <typename E>
  QMOE_DEV float get(int i) const {
    if constexpr (BYTES == 4) return __uint_as_float(w[i]);
    else return E::load((uint16_t)(w[i / 2] >> (16 * (i & 1))));
  }
};

static inline bool known_type(int t) { return t == QMOE_BF16 || t == QMOE_F16 || t == QMOE_F32; }
