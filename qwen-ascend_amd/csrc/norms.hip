// Norms around a block: the RMS norm before it, and what follows it (its norm, gate and
// residual scale, the residual sum, the next norm).
//
//   n(v; w) = v * (mean(v^2) + eps)^(-1/2) * (offset + w)          per row of H
//   p = n(y; post) or y;  h = r + scale * a(gate) * p;  x = n(h; next)
//
// All of it in fp32 with one rounding per output; x is normed from h before h's rounding.
#include "elem_types.h"

#include <algorithm>
#include <cmath>

namespace {

struct NormArgs {
  const void* y;      // block output, or null: h = r
  const void* r;      // residual
  const void* post;   // weight of the norm of y, or null
  const void* gate;   // or null
  const void* next;   // weight of the norm of h, or null
  void* h;            // or null
  void* x;            // or null
  long ldy, ldr, ldg, ldh, ldx, rows;
  int H, gate_step;   // gate column step: 0 (one value per row) or 1
  int post_type, gate_type, next_type, gate_sigmoid;
  float scale, eps, offset;
};

constexpr int THREADS = 256, WAVES = THREADS / 64;

template <typename V>
QMOE_DEV V block_sum(V v, V* lds) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  V s = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) s += lds[w];
  return s;
}

// (pre, r) with v * pre * r = v * (mean(v^2) + eps)^(-1/2). A sum of squares that leaves
// the fp32 range is taken again in 64 bits, where pre keeps r a normal number.
struct Rms {
  float pre, r;
};
template <typename F>
QMOE_DEV Rms row_rms(F value, int H, float eps) {
  __shared__ float lds[WAVES];
  __shared__ double lds64[WAVES];
  float s = 0.f;
  for (int i = threadIdx.x; i < H; i += THREADS) {
    const float v = value(i);
    s += v * v;
  }
  s = block_sum(s, lds);
  if (s <= 3.402823466e38f) return {1.f, 1.f / sqrtf(s / (float)H + eps)};
  double d = 0.0;
  for (int i = threadIdx.x; i < H; i += THREADS) {
    const double v = value(i);
    d += v * v;
  }
  d = block_sum(d, lds64);
  return {0x1p-60f, (float)(0x1p60 / sqrt(d / H + eps))};
}

template <typename Y, typename R>
__global__ __launch_bounds__(THREADS) void norm_rows_kernel(NormArgs a) {
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const auto* y = static_cast<const typename Y::raw*>(a.y) + row * a.ldy;
    const auto* r = static_cast<const typename R::raw*>(a.r) + row * a.ldr;
    Rms post = {1.f, 1.f}, next = {1.f, 1.f};
    if (a.post) post = row_rms([&](int i) { return Y::load(y[i]); }, a.H, a.eps);
    auto sum = [&](int i) {
      float h = R::load(r[i]);
      if (!a.y) return h;
      float p = Y::load(y[i]);
      if (a.post) p = p * post.pre * post.r * (a.offset + load_typed(a.post, i, a.post_type));
      float g = a.scale;
      if (a.gate) {
        float v = load_typed(a.gate, row * a.ldg + (long)i * a.gate_step, a.gate_type);
        if (a.gate_sigmoid) v = 1.f / (1.f + expf(-v));
        g *= v;
      }
      return h + g * p;
    };
    if (a.next) next = row_rms(sum, a.H, a.eps);
    __syncthreads();  // h may overwrite r: every read of the row's sums above comes first
    for (int i = threadIdx.x; i < a.H; i += THREADS) {
      const float h = sum(i);
      if (a.h) static_cast<typename R::raw*>(a.h)[row * a.ldh + i] = R::store(h);
      if (a.next)
        static_cast<typename Y::raw*>(a.x)[row * a.ldx + i] =
            Y::store(h * next.pre * next.r * (a.offset + load_typed(a.next, i, a.next_type)));
    }
  }
}

template <typename Y, typename R>
int launch(const NormArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((norm_rows_kernel<Y, R>), dim3((unsigned)std::min<long>(a.rows, 1 << 20)), dim3(THREADS), 0, st, a);
  return (int)hipGetLastError();
}

// 16-bit block types with a residual of the same type or of 32 bits, or all in 32 bits.
int dispatch(const NormArgs& a, int ytype, int rtype, hipStream_t st) {
  if (ytype == QMOE_BF16 && rtype == QMOE_BF16) return launch<ElemBF16, ElemBF16>(a, st);
  if (ytype == QMOE_BF16 && rtype == QMOE_F32) return launch<ElemBF16, ElemF32>(a, st);
  if (ytype == QMOE_F16 && rtype == QMOE_F16) return launch<ElemF16, ElemF16>(a, st);
  if (ytype == QMOE_F16 && rtype == QMOE_F32) return launch<ElemF16, ElemF32>(a, st);
  if (ytype == QMOE_F32 && rtype == QMOE_F32) return launch<ElemF32, ElemF32>(a, st);
  return QMOE_EINVAL;
}

// Longest row, and the smallest eps against which the squares that fp32 loses
// below its range are nothing.
constexpr int H_MAX = 32768;
constexpr float EPS_MIN = 1e-30f;

bool bad_scalars(int H, float eps, float offset, float scale) {
  return H < 1 || H > H_MAX || !(eps >= EPS_MIN) || !std::isfinite(eps) || !std::isfinite(offset) ||
         !std::isfinite(scale);
}

}  // namespace

extern "C" {

int qmoe_block_norm(const void* x, long ldx, int xtype, const void* weight, int wtype, void* y, long ldy, int ytype,
                    long rows, int H, float eps, float offset, void* stream) {
  if (rows < 0 || bad_scalars(H, eps, offset, 1.f) || !known_type(wtype) || ldx < 0 || ldy < H) return QMOE_EINVAL;
  if (rows == 0) return QMOE_OK;
  if (!x || !weight || !y) return QMOE_EINVAL;
  NormArgs a = {};
  a.r = x, a.ldr = ldx, a.next = weight, a.next_type = wtype, a.x = y, a.ldx = ldy;
  a.rows = rows, a.H = H, a.eps = eps, a.offset = offset, a.scale = 1.f;
  return dispatch(a, ytype, xtype, (hipStream_t)stream);
}

int qmoe_block_residual(const void* y, long ldy, int ytype, const void* residual, long ldr, int rtype,
                        const void* post_weight, int post_type, const void* gate, long gate_row_step,
                        int gate_column_step, int gate_type, int gate_sigmoid, float scale, void* h, long ldh,
                        const void* next_weight, int next_type, void* x, long ldx, long rows, int H, float eps,
                        float offset, void* stream) {
  if (rows < 0 || bad_scalars(H, eps, offset, scale) || ldy < 0 || ldr < 0 || ldh < H) return QMOE_EINVAL;
  if (post_weight && !known_type(post_type)) return QMOE_EINVAL;
  if (gate && (!known_type(gate_type) || gate_row_step < 0 || (gate_column_step != 0 && gate_column_step != 1)))
    return QMOE_EINVAL;
  if ((next_weight == nullptr) != (x == nullptr) || (next_weight && (!known_type(next_type) || ldx < H)))
    return QMOE_EINVAL;
  if (rows == 0) return QMOE_OK;
  if (!y || !residual || !h || (h == residual && ldh != ldr)) return QMOE_EINVAL;
  NormArgs a = {};
  a.y = y, a.ldy = ldy, a.r = residual, a.ldr = ldr, a.h = h, a.ldh = ldh;
  a.post = post_weight, a.post_type = post_type;
  a.gate = gate, a.ldg = gate_row_step, a.gate_step = gate_column_step, a.gate_type = gate_type;
  a.gate_sigmoid = gate_sigmoid;
  a.next = next_weight, a.next_type = next_type, a.x = x, a.ldx = ldx;
  a.rows = rows, a.H = H, a.eps = eps, a.offset = offset, a.scale = scale;
  return dispatch(a, ytype, rtype, (hipStream_t)stream);
}

}  // extern "C"
