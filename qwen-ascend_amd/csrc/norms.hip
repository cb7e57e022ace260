// Norms around a block: the RMS norm before it, and what follows it (its norm, gate and
// residual scale, the residual sum, the next norm).
//
//   n(v; w) = v * (mean(v^2) + eps)^(-1/2) * (offset + w)          per row of H
//   p = n(y; post) or y;  h = r + scale * a(gate) * p;  x = n(h; next)
//
// All of it in fp32 with one rounding per output; x is normed from h before h's rounding.
#include "elem_types.h"

#include <algorithm>
#include <cfloat>
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

// Memory bound: each operand is read once and each output written once. A row belongs to a
// workgroup (or, where it is short, to one wave, four rows per workgroup and no barrier); each
// thread holds NV pieces of 16 bytes of y in registers from the load to the last store, and a
// workgroup with more than one row loads the next one while it works on this one.
// 4096 x 2560 bf16: 10.9 us for the norm (42 MB), 20.8 for the whole step after a block (84
// MB); copies of the same bytes take 10.0 and 17.7. 8192 x 4096 with a 32-bit stream: 77.9 us,
// 5.2 TB/s.
template <typename Y>
constexpr int VE = 16 / sizeof(typename Y::raw);

template <typename T>
QMOE_DEV T wave_sum(T v) {
  if constexpr (sizeof(T) == 4) return wave_sum_f32(v);
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// LDS writes before it are seen after it; global loads and stores stay in flight.
QMOE_DEV void barrier_lds() {
  asm volatile("" ::: "memory");
  wait_vm_lgkm0<63>();
  barrier_no_fence();
}

template <bool ONE_WAVE, typename T>
QMOE_DEV T row_sum(T v, T* lds, int waves) {
  v = wave_sum(v);
  if constexpr (ONE_WAVE) return v;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  barrier_lds();
  T s = lds[0];
  for (int w = 1; w < waves; ++w) s += lds[w];
  return s;
}

// (pre, r) with v * pre * r = v * (mean(v^2) + eps)^(-1/2). A sum of squares that leaves the
// fp32 range is taken again in 64 bits, where pre keeps r a normal number.
struct Rms {
  float pre, r;
};
template <bool ONE_WAVE, int N>
QMOE_DEV Rms row_rms(const float (&v)[N], int H, float eps, float* lds, double* lds64, int waves) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) s += v[i] * v[i];
  s = row_sum<ONE_WAVE>(s, lds, waves);
  if (s <= FLT_MAX) return {1.f, 1.f / sqrtf(s / (float)H + eps)};
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) d += (double)v[i] * v[i];
  d = row_sum<ONE_WAVE>(d, lds64, waves);
  return {0x1p-60f, (float)(0x1p60 / sqrt(d / H + eps))};
}

// N elements of a tensor whose type is known at run time only.
template <int N>
struct AnyVec {
  RawVec<N, 4> v;
  QMOE_DEV void load(const void* p, long at, int type) {
    if (type == QMOE_F32) {
      v.load(static_cast<const float*>(p) + at);
    } else {
      RawVec<N, 2> h;
      h.load(static_cast<const uint16_t*>(p) + at);
#pragma unroll
      for (int i = 0; i < h.WORDS; ++i) v.w[i] = h.w[i];
    }
  }
  // Unpacked again at each use: the compiler would keep the 32-bit values over the whole loop
  // otherwise.
  QMOE_DEV void pin() {
#pragma unroll
    for (int i = 0; i < v.WORDS; ++i) asm volatile("" : "+v"(v.w[i]));
  }
  QMOE_DEV void unpack(float (&f)[N], int type) const {
    if (type == QMOE_F32) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = __uint_as_float(v.w[i]);
    } else if (type == QMOE_BF16) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = ElemBF16::load((uint16_t)(v.w[i / 2] >> (16 * (i & 1))));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = ElemF16::load((uint16_t)(v.w[i / 2] >> (16 * (i & 1))));
    }
  }
};

QMOE_DEV float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + expf(-v)); }

template <typename E, int N>
QMOE_DEV void store_piece(const float* f, typename E::raw* p) {
  RawVec<N, sizeof(typename E::raw)> o;
  if constexpr (sizeof(typename E::raw) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) o.w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) o.w[i / 2] = E::pack(f[i], f[i + 1]);
  }
  o.store(p);
}

// What a call does: the norm alone; a residual sum whose gate is one value per row (or
// none); one whose gate has a value per element (or channel).
enum { NORM, SUM, SUM_GATED };

// One row's operands as loaded: whole pieces, and the one element of the row's end.
template <typename Y, typename R, int NV, int MODE>
struct RowIn {
  static constexpr int N = VE<Y>;
  RawVec<N, sizeof(typename Y::raw)> y[MODE == NORM ? 1 : NV];
  RawVec<N, sizeof(typename R::raw)> r[NV];
  AnyVec<N> g[MODE == SUM_GATED ? NV : 1];
  float y_end, r_end, g_end;

  QMOE_DEV void load(const NormArgs& a, long row, int tpr, int tid, int whole) {
    const auto* yp = static_cast<const typename Y::raw*>(a.y) + row * a.ldy;
    const auto* rp = static_cast<const typename R::raw*>(a.r) + row * a.ldr;
    const long gp = row * a.ldg;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * tpr + tid) * N;
      r[j].zero();
      if constexpr (MODE != NORM) y[j].zero();
      if constexpr (MODE == SUM_GATED) g[j].v.zero();
      if (c < whole) {
        r[j].load(rp + c);
        if constexpr (MODE != NORM) y[j].load(yp + c);
        if constexpr (MODE == SUM_GATED) g[j].load(a.gate, gp + c, a.gate_type);
      }
    }
    y_end = r_end = g_end = 0.f;
    const int last = whole + tid;
    if (last < a.H) {
      r_end = R::load(rp[last]);
      if constexpr (MODE != NORM) y_end = Y::load(yp[last]);
      if constexpr (MODE == SUM_GATED) g_end = load_typed(a.gate, gp + last, a.gate_type);
    }
    if constexpr (MODE == SUM)
      if (a.gate) g_end = load_typed(a.gate, gp, a.gate_type);
  }
};

// offset + weight for this thread's places; loaded once for all its rows.
template <int NV, int N>
struct Weights {
  AnyVec<N> w[NV];
  float end;
  QMOE_DEV void load(const void* p, int type, int H, int tpr, int tid, int whole) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * tpr + tid) * N;
      w[j].v.zero();
      if (c < whole) w[j].load(p, c, type);
    }
    end = whole + tid < H ? load_typed(p, whole + tid, type) : 0.f;
  }
  // v = v * m * (offset + w)
  QMOE_DEV void apply(float (&v)[NV * N + 1], const Rms m, float offset, int type) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[N];
      w[j].pin();
      w[j].unpack(f, type);
#pragma unroll
      for (int i = 0; i < N; ++i) v[j * N + i] = v[j * N + i] * m.pre * m.r * (offset + f[i]);
    }
    v[NV * N] = v[NV * N] * m.pre * m.r * (offset + end);
  }
};

template <typename E, int NV, int N>
QMOE_DEV void store_row(const float (&v)[NV * N + 1], typename E::raw* p, int H, int tpr, int tid, int whole) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * tpr + tid) * N;
    if (c < whole) store_piece<E, N>(v + j * N, p + c);
  }
  if (whole + tid < H) p[whole + tid] = E::store(v[NV * N]);
}

// Places behind the row hold zeros and stay zero through all of it (or turn NaN only where a
// row's scale factors are infinite or NaN, with the whole row).
template <typename Y, typename R, int NV, int MODE, int MAX_WAVES, bool AHEAD>
__global__ __launch_bounds__(MAX_WAVES == 1 ? 256 : 64 * MAX_WAVES) void norm_rows_kernel(NormArgs a) {
  constexpr bool ONE_WAVE = MAX_WAVES == 1;
  constexpr int N = VE<Y>, L = NV * N;
  __shared__ float lds[2][16];
  __shared__ double lds64[2][16];
  const int tpr = ONE_WAVE ? 64 : blockDim.x, waves = tpr / 64;
  const int tid = ONE_WAVE ? threadIdx.x & 63 : threadIdx.x;
  const long step = ONE_WAVE ? gridDim.x * 4l : gridDim.x;
  const int whole = a.H / N * N;
  long row = ONE_WAVE ? blockIdx.x * 4l + (threadIdx.x >> 6) : blockIdx.x;
  if (row >= a.rows) return;
  RowIn<Y, R, NV, MODE> in;
  Weights<NV, N> post, next;
  in.load(a, row, tpr, tid, whole);
  if (MODE != NORM && a.post) post.load(a.post, a.post_type, a.H, tpr, tid, whole);
  if (a.next) next.load(a.next, a.next_type, a.H, tpr, tid, whole);
  for (;;) {
    const long following = row + step;
    RowIn<Y, R, NV, MODE> ahead;
    if (AHEAD && following < a.rows) ahead.load(a, following, tpr, tid, whole);
    float v[L + 1];
    if constexpr (MODE == NORM) {
#pragma unroll
      for (int i = 0; i < L; ++i) v[i] = in.r[i / N].template get<R>(i % N);
      v[L] = in.r_end;
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i) v[i] = in.y[i / N].template get<Y>(i % N);
      v[L] = in.y_end;
      if (a.post) post.apply(v, row_rms<ONE_WAVE>(v, a.H, a.eps, lds[0], lds64[0], waves), a.offset, a.post_type);
      float scale = a.scale;
      if constexpr (MODE == SUM) {
        if (a.gate) scale *= a.gate_sigmoid ? sigmoid(in.g_end) : in.g_end;
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float g[N];
          in.g[j].unpack(g, a.gate_type);
          if (a.gate_sigmoid) {
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = sigmoid(g[i]);
          }
#pragma unroll
          for (int i = 0; i < N; ++i) v[j * N + i] *= g[i];
        }
        v[L] *= a.gate_sigmoid ? sigmoid(in.g_end) : in.g_end;
      }
#pragma unroll
      for (int i = 0; i < L; ++i) v[i] = in.r[i / N].template get<R>(i % N) + scale * v[i];
      v[L] = in.r_end + scale * v[L];
      store_row<R, NV, N>(v, static_cast<typename R::raw*>(a.h) + row * a.ldh, a.H, tpr, tid, whole);
    }
    if (a.next) {
      next.apply(v, row_rms<ONE_WAVE>(v, a.H, a.eps, lds[1], lds64[1], waves), a.offset, a.next_type);
      store_row<Y, NV, N>(v, static_cast<typename Y::raw*>(a.x) + row * a.ldx, a.H, tpr, tid, whole);
    }
    if (following >= a.rows) break;
    row = following;
    if constexpr (AHEAD) in = ahead;
    else in.load(a, row, tpr, tid, whole);
    if constexpr (!ONE_WAVE) barrier_lds();  // the next row's sums reuse the LDS slots
  }
}

// Rows longer than a workgroup's registers hold: each pass over the row reads it again.
constexpr int WIDE_THREADS = 1024;
template <typename F>
QMOE_DEV Rms wide_rms(F value, int H, float eps, float* lds, double* lds64) {
  float s = 0.f;
  for (int i = threadIdx.x; i < H; i += WIDE_THREADS) {
    const float v = value(i);
    s += v * v;
  }
  s = row_sum<false>(s, lds, WIDE_THREADS / 64);
  if (s <= FLT_MAX) return {1.f, 1.f / sqrtf(s / (float)H + eps)};
  double d = 0.0;
  for (int i = threadIdx.x; i < H; i += WIDE_THREADS) {
    const double v = value(i);
    d += v * v;
  }
  d = row_sum<false>(d, lds64, WIDE_THREADS / 64);
  return {0x1p-60f, (float)(0x1p60 / sqrt(d / H + eps))};
}

template <typename Y, typename R>
__global__ __launch_bounds__(WIDE_THREADS) void norm_wide_kernel(NormArgs a) {
  __shared__ float lds[2][16];
  __shared__ double lds64[2][16];
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const auto* y = static_cast<const typename Y::raw*>(a.y) + row * a.ldy;
    const auto* r = static_cast<const typename R::raw*>(a.r) + row * a.ldr;
    Rms post = {1.f, 1.f}, next = {1.f, 1.f};
    if (a.post) post = wide_rms([&](int i) { return Y::load(y[i]); }, a.H, a.eps, lds[0], lds64[0]);
    auto sum = [&](int i) {
      const float res = R::load(r[i]);
      if (!a.y) return res;
      float p = Y::load(y[i]);
      if (a.post) p = p * post.pre * post.r * (a.offset + load_typed(a.post, i, a.post_type));
      float scale = a.scale;
      if (a.gate) {
        const float g = load_typed(a.gate, row * a.ldg + (long)i * a.gate_step, a.gate_type);
        scale *= a.gate_sigmoid ? sigmoid(g) : g;
      }
      return res + scale * p;
    };
    if (a.next) next = wide_rms(sum, a.H, a.eps, lds[1], lds64[1]);
    for (int i = threadIdx.x; i < a.H; i += WIDE_THREADS) {  // h may overwrite r: each place by its own thread
      const float h = sum(i);
      if (a.h) static_cast<typename R::raw*>(a.h)[row * a.ldh + i] = R::store(h);
      if (a.next)
        static_cast<typename Y::raw*>(a.x)[row * a.ldx + i] =
            Y::store(h * next.pre * next.r * (a.offset + load_typed(a.next, i, a.next_type)));
    }
    barrier_lds();
  }
}

template <typename Y, typename R, int NV, int MODE, int MAX_WAVES, bool AHEAD>
int launch_rows(const NormArgs& a, int waves, hipStream_t st) {
  // With rows ahead: as many workgroups as stay resident with 16 waves per CU, the rows in
  // even rounds over them (4096 x 2560 norm: 10.9 us; 12 waves 13.0, 20 waves 11.0). The
  // others take a row each and leave the order to the dispatcher.
  const int rows_per = MAX_WAVES == 1 ? 4 : 1, wg_waves = MAX_WAVES == 1 ? 4 : waves;
  const long groups = (a.rows + rows_per - 1) / rows_per, most = AHEAD ? 256l * (16 / wg_waves) : 1l << 20;
  const long rounds = (groups + most - 1) / most;
  const unsigned grid = (unsigned)((groups + rounds - 1) / rounds);
  hipLaunchKernelGGL((norm_rows_kernel<Y, R, NV, MODE, MAX_WAVES, AHEAD>), dim3(grid), dim3(64 * wg_waves), 0, st, a);
  return (int)hipGetLastError();
}

// Few rows: one piece per thread and the whole row in flight at once (1 x 2048: 2.3 us in a
// graph, 2.4 to 2.5 with two pieces; 4 x 2560 sum 3.6 and 3.8). More of them: up to two pieces
// per thread, so that a row takes half the waves (4096 x 2560 sum: 20.8 us, one piece 23.9;
// 8192 x 1536: 22.8 and 24.0), and the next row on its way, where the registers hold it: not for
// 16 waves with 32-bit sums or a gate per element (2048 x 16384 sum in bf16: 59.9 us, without
// the row ahead 68.1; in fp16, with nine words spilled, 66.0 and 70.4).
template <typename Y, typename R, int MODE>
int launch_mode(const NormArgs& a, hipStream_t st) {
  const int pieces = host_ceil_div(a.H, VE<Y>);
  auto waves = [&](int nv) { return host_ceil_div(pieces, 64 * nv); };
  if (a.rows <= 512) {
    if (waves(1) <= 16) return launch_rows<Y, R, 1, MODE, 16, false>(a, waves(1), st);
  } else {
    if (waves(1) == 1) return launch_rows<Y, R, 1, MODE, 1, true>(a, 1, st);
    if (waves(2) == 1) return launch_rows<Y, R, 2, MODE, 1, true>(a, 1, st);
    if (waves(2) <= 8) return launch_rows<Y, R, 2, MODE, 8, true>(a, waves(2), st);
    if constexpr (MODE == NORM || (MODE == SUM && sizeof(typename R::raw) == 2))
      if (waves(2) <= 16) return launch_rows<Y, R, 2, MODE, 16, true>(a, waves(2), st);
  }
  if (waves(2) <= 16) return launch_rows<Y, R, 2, MODE, 16, false>(a, waves(2), st);
  if constexpr (VE<Y> == 4)
    if (waves(4) <= 16) return launch_rows<Y, R, 4, MODE, 16, false>(a, waves(4), st);
  hipLaunchKernelGGL((norm_wide_kernel<Y, R>), dim3((unsigned)std::min<long>(a.rows, 1 << 20)), dim3(WIDE_THREADS), 0, st,
                     a);
  return (int)hipGetLastError();
}

template <typename Y, typename R>
int launch(const NormArgs& a, hipStream_t st) {
  if (!a.y) return launch_mode<Y, R, NORM>(a, st);
  if (a.gate && a.gate_step) return launch_mode<Y, R, SUM_GATED>(a, st);
  return launch_mode<Y, R, SUM>(a, st);
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
