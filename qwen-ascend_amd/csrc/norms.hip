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
// 5.2 TB/s. All in fp32: norm 4096 x 2560 15.9 us, 5.3 TB/s, 2048 x 16384 53 us, 5.0 TB/s; the whole
// step, gate per row 40.8 and 114 us, 4.1 and 4.7 TB/s, gate per element 55.2 and 188 us.
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
template <typename T, int N>
QMOE_DEV T squares(const float (&v)[N]) {
  T s = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) s += (T)v[i] * (T)v[i];
  return s;
}
// mine(T()): the squares of this thread's places in T
template <bool ONE_WAVE, typename F>
QMOE_DEV Rms rms_of(F mine, int H, float eps, float* lds, double* lds64, int waves) {
  const float s = row_sum<ONE_WAVE>(mine(0.f), lds, waves);
  if (s <= FLT_MAX) return {1.f, 1.f / sqrtf(s / (float)H + eps)};
  const double d = row_sum<ONE_WAVE>(mine(0.0), lds64, waves);
  return {0x1p-60f, (float)(0x1p60 / sqrt(d / H + eps))};
}
template <bool ONE_WAVE, int N>
QMOE_DEV Rms row_rms(const float (&v)[N], int H, float eps, float* lds, double* lds64, int waves) {
  return rms_of<ONE_WAVE>([&](auto zero) { return squares<decltype(zero)>(v); }, H, eps, lds, lds64, waves);
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

  // Pieces from column `begin` on; the row's last elements with them where `ends`.
  QMOE_DEV void load(const NormArgs& a, long row, int tpr, int tid, int whole, int begin = 0, bool ends = true) {
    const auto* yp = static_cast<const typename Y::raw*>(a.y) + row * a.ldy;
    const auto* rp = static_cast<const typename R::raw*>(a.r) + row * a.ldr;
    const long gp = row * a.ldg;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = begin + (j * tpr + tid) * N;
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
    if (ends && last < a.H) {
      r_end = R::load(rp[last]);
      if constexpr (MODE != NORM) y_end = Y::load(yp[last]);
      if constexpr (MODE == SUM_GATED) g_end = load_typed(a.gate, gp + last, a.gate_type);
    }
    if constexpr (MODE == SUM)
      if (a.gate) g_end = load_typed(a.gate, gp, a.gate_type);
  }

  // What is normed first: y, or the residual where there is no y.
  QMOE_DEV void unpack(float (&v)[NV * N + 1]) const {
#pragma unroll
    for (int i = 0; i < NV * N; ++i) {
      if constexpr (MODE == NORM) v[i] = r[i / N].template get<R>(i % N);
      else v[i] = y[i / N].template get<Y>(i % N);
    }
    v[NV * N] = MODE == NORM ? r_end : y_end;
  }

  // v, the block's (normed) output, becomes r + scale * a(gate) * v.
  QMOE_DEV void sum(const NormArgs& a, float (&v)[NV * N + 1]) const {
    float scale = a.scale;
    if constexpr (MODE == SUM) {
      if (a.gate) scale *= a.gate_sigmoid ? sigmoid(g_end) : g_end;
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float f[N];
        g[j].unpack(f, a.gate_type);
        if (a.gate_sigmoid) {
#pragma unroll
          for (int i = 0; i < N; ++i) f[i] = sigmoid(f[i]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) v[j * N + i] *= f[i];
      }
      v[NV * N] *= a.gate_sigmoid ? sigmoid(g_end) : g_end;
    }
#pragma unroll
    for (int i = 0; i < NV * N; ++i) v[i] = r[i / N].template get<R>(i % N) + scale * v[i];
    v[NV * N] = r_end + scale * v[NV * N];
  }
};

// offset + weight for this thread's places; loaded once for all its rows.
template <int NV, int N>
struct Weights {
  AnyVec<N> w[NV];
  float end;
  QMOE_DEV void load(const void* p, int type, int H, int tpr, int tid, int whole, int begin = 0, bool ends = true) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = begin + (j * tpr + tid) * N;
      w[j].v.zero();
      if (c < whole) w[j].load(p, c, type);
    }
    end = ends && whole + tid < H ? load_typed(p, whole + tid, type) : 0.f;
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
QMOE_DEV void store_row(const float (&v)[NV * N + 1], typename E::raw* p, int H, int tpr, int tid, int whole, int begin = 0,
                        bool ends = true) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = begin + (j * tpr + tid) * N;
    if (c < whole) store_piece<E, N>(v + j * N, p + c);
  }
  if (ends && whole + tid < H) p[whole + tid] = E::store(v[NV * N]);
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
    in.unpack(v);
    if constexpr (MODE != NORM) {
      if (a.post) post.apply(v, row_rms<ONE_WAVE>(v, a.H, a.eps, lds[0], lds64[0], waves), a.offset, a.post_type);
      in.sum(a, v);
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

// Rows longer than a workgroup's registers hold: the same in steps of a piece per thread, each
// pass over the row reading it again (from the caches; 2048 x 32768 bf16: norm 62.9 us, 4.3 TB/s,
// the whole step after a block 157 us, 3.4 TB/s).
constexpr int WIDE_THREADS = 1024;
template <typename Y, typename R, int MODE>
__global__ __launch_bounds__(WIDE_THREADS) void norm_wide_kernel(NormArgs a) {
  constexpr int N = VE<Y>, SPAN = WIDE_THREADS * N, WAVES = WIDE_THREADS / 64;
  __shared__ float lds[2][WAVES];
  __shared__ double lds64[2][WAVES];
  const int tid = threadIdx.x, whole = a.H / N * N;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    RowIn<Y, R, 1, MODE> in;
    Weights<1, N> w;
    float v[N + 1];
    Rms post = {1.f, 1.f};
    auto each = [&](auto f) {
      for (int c = 0; c < whole; c += SPAN) {
        const bool ends = c + SPAN >= whole;
        in.load(a, row, WIDE_THREADS, tid, whole, c, ends);
        in.unpack(v);
        f(c, ends);
      }
    };
    auto sum = [&](int c, bool ends) {
      if constexpr (MODE != NORM) {
        if (a.post) {
          w.load(a.post, a.post_type, a.H, WIDE_THREADS, tid, whole, c, ends);
          w.apply(v, post, a.offset, a.post_type);
        }
        in.sum(a, v);
      }
    };
    if (MODE != NORM && a.post)
      post = rms_of<false>([&](auto s) {
        each([&](int, bool) { s += squares<decltype(s)>(v); });
        return s;
      }, a.H, a.eps, lds[0], lds64[0], WAVES);
    Rms next = {1.f, 1.f};
    if (a.next)
      next = rms_of<false>([&](auto s) {
        each([&](int c, bool ends) {
          sum(c, ends);
          s += squares<decltype(s)>(v);
        });
        return s;
      }, a.H, a.eps, lds[1], lds64[1], WAVES);
    each([&](int c, bool ends) {  // h may overwrite r: each place read and written by one thread
      sum(c, ends);
      if constexpr (MODE != NORM)
        store_row<R, 1, N>(v, static_cast<typename R::raw*>(a.h) + row * a.ldh, a.H, WIDE_THREADS, tid, whole, c, ends);
      if (a.next) {
        w.load(a.next, a.next_type, a.H, WIDE_THREADS, tid, whole, c, ends);
        w.apply(v, next, a.offset, a.next_type);
        store_row<Y, 1, N>(v, static_cast<typename Y::raw*>(a.x) + row * a.ldx, a.H, WIDE_THREADS, tid, whole, c, ends);
      }
    });
    barrier_lds();
  }
}

template <typename Y, typename R, int NV, int MODE, int MAX_WAVES, bool AHEAD>
int launch_rows(const NormArgs& a, int waves, hipStream_t st) {
  // With rows ahead: as many workgroups as 16 waves per CU make, the rows in even rounds over
  // them. That is what stays resident up to 128 registers. Above, fewer do, and part of the
  // grid waits: 12 waves with a gate per row in fp16 (137 to 140), in bf16 with rows of one wave
  // (130) and beside fp32 (153 to 156), and with one per element in bf16 (164), 8 with one per
  // element in fp16 (170) and beside fp32 (186 to 189). Grids of 8, 12, 16 and 20
  // waves, us: 4096 x 2560 norm 13.0, 10.0, 10.0, 10.1; bf16 sum, gate per row 24.7, 18.8, 18.8,
  // 20.3; per channel beside fp32 33.4, 34.7, 34.6, 37.8; 8192 x 4096, gate per element fp16
  // 65.9, 73.3, 65.4, 71.9, beside fp32 88.9, 103, 89.0, 96.7. Against 16 stand rows of two and
  // of eight waves beside fp32: 8192 x 1536 per channel 34.6, 45.5, 42.6, 42.6, 3000 x 8192 62.9,
  // 62.8, 65.4, 65.2. The other forms take a row each and leave the order to the dispatcher.
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
// Where few rows end depends on the form; 512 is one limit for all. One piece and two with the
// row ahead, us:
//   norm bf16                400 x 4096   4.1 /  4.0     1003 x 2048  4.1 /  4.1    1003 x 4096   5.9 /  5.6
//   sum, gate per row, bf16  400 x 2048   4.9 /  5.2      513 x 2048  5.3 /  5.6    2048 x 4096  15.1 / 13.5
//   gate per element, fp16   400 x 2048   5.2 /  6.4      777 x 2048  7.4 /  7.6    1003 x 2048   7.9 /  8.1
//                           2048 x 2048  11.7 / 13.9     4096 x 2048 17.4 / 23.2    2048 x 8192  45.6 / 40.9
//   per channel beside fp32  400 x 2048   5.5 /  6.5     2048 x 2048 14.3 / 17.9    2048 x 8192  55.0 / 46.3
//   gate per row, fp16      1003 x 2048   6.8 /  6.8     4096 x 2048 13.6 / 16.4    2048 x 4096  15.4 / 15.8
// So two pieces win from the limit on for norms, for a gate per row in bf16 and for rows of 8192, but not for
// rows of 2048 in fp16 or under a gate per element or channel, which lose up to a quarter there, nor for rows
// of 4096 in fp16 or per channel beside fp32 (up to a seventh); with up to two rows per workgroup the row ahead
// is hardly ever loaded. Below the limit rows of 8192 under a gate per row in bf16 lose a quarter (400: 10.9 / 8.4).
// Forms that spill: a gate per element on 16 waves in fp32 with four pieces, 24 words (2048 x 16384:
// 188 us, 3.6 TB/s; a gate per row, without spills, 114 us, 4.7), fp16 beside fp32 4 words and bf16
// beside fp32 1 (117 and 112 us, 4.0 and 4.2 TB/s; a gate per row 96 us, 4.2).
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
  hipLaunchKernelGGL((norm_wide_kernel<Y, R, MODE>), dim3((unsigned)std::min<long>(a.rows, 1 << 20)), dim3(WIDE_THREADS),
                     0, st, a);
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
