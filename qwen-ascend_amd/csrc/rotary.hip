// Rotary positions, alone and on the way into a paged cache.
//
// Pair i of a head at position p turns by the angle 2 pi p f_i, f_i in turns per position:
//   (a, b) -> turn * (a cos - b sin, b cos + a sin)
// Pairs are (x_i, x_{i + rd/2}) or (x_2i, x_{2i+1}), i < rd/2; elements from rd on are copied.
//
// Frequencies come as 64-bit fractions of a turn, so that p f_i mod 1 is one integer product, exact
// at any position (the frequency itself is rounded once, to 53 bits where it was worked out in double
// precision); its leading 32 bits are the angle (2^-32 of a turn), and cosine and sine are
// taken of it in fp32, where the angle in half turns keeps 24 bits: fp32 outputs are off by 4.3e-8 of their norm,
// with angles and their functions in 64 bits 3.3e-8. One rounding per output.
#include "paged.h"

#include <algorithm>

namespace {

constexpr int D_MAX = 1024;
constexpr unsigned GRID_X = 1 << 20;  // workgroups in a row of the grid: a dimension's threads are counted in 32 bits

struct HeadRows {  // rows [T, heads, D]: element steps of a token and of a head
  const void* p;
  long token, head;
};

struct RotateArgs {
  HeadRows q, k, v;
  void* q_out;
  long out_token, out_head;
  void *k_cache, *v_cache;
  CacheSteps kc, vc;
  Batch batch;
  const uint64_t* frequencies;
  const void* positions;
  int positions64, interleaved;
  int Hq, Hkv, heads;  // heads: of a token, queries first, then keys and values
  int D, rd, turned;   // turned: items of a head that turn
  int per_unit, units;
  FastDiv items, groups;  // items of a head; units of a token
  float turn;
};

// C consecutive elements.
template <typename E, int C>
struct Chunk {
  using raw = typename E::raw;
  raw e[C];
  QMOE_DEV void load(const raw* p) {
    if constexpr (C * sizeof(raw) == 16) {
      const u32x4_any v = *reinterpret_cast<const u32x4_any*>(p);
      __builtin_memcpy(e, &v, 16);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) e[i] = p[i];
    }
  }
  QMOE_DEV void store(raw* p) const {
    if constexpr (C * sizeof(raw) == 16) {
      u32x4_any v;
      __builtin_memcpy(&v, e, 16);
      *reinterpret_cast<u32x4_any*>(p) = v;
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) p[i] = e[i];
    }
  }
};

// (a cos - b sin, b cos + a sin), with one rounding order for all forms of the kernel: a head's bits then do not
// depend on how many tokens a call has.
QMOE_DEV void turn_pair(float& a, float& b, float c, float s) {
  const float as = a * s;
  a = __builtin_fmaf(a, c, -(b * s));
  b = __builtin_fmaf(b, c, as);
}

// Memory bound: each element is read and written once. A wave takes one token and up to
// U x 64 items of its heads, an item being two chunks of C elements that turn together (or are
// copied); it has all its loads in flight while it works out the token's angles, a pair per lane,
// which its lanes then share through LDS.
// 8192 tokens of 16 heads of 256, 64 elements turned, 134 MB: 22.4 us, 6.0 TB/s (caches included); 2246 tokens of
// 32 + 16 heads of 128 into a cache, 55 MB: 14.2 us, 3.9 TB/s, as a token's place is looked up before its
// stores. Few tokens by launch and latency: one of 32 heads 2.9 us, 64 of 32 + 8 into a cache 4.5.
template <typename E, int C, int U>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a) {
  using raw = typename E::raw;
  __shared__ float cosine[4][D_MAX / 2], sine[4][D_MAX / 2];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const unsigned unit = (blockIdx.y * GRID_X + blockIdx.x) * 4 + wave;
  if (unit >= (unsigned)a.units) return;
  const int t = a.groups.div(unit), first = ((int)unit - t * (int)a.groups.d) * a.per_unit;
  const int count = min(a.per_unit, a.heads - first) * (int)a.items.d;

  Chunk<E, C> x[U], y[U];
  int head[U], item[U], at[U], then[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = lane + 64 * u, h = a.items.div(i);
    head[u] = i < count ? first + h : -1;
    item[u] = i - h * (int)a.items.d;
    const bool turns = item[u] < a.turned, apart = turns && !a.interleaved;
    at[u] = apart ? item[u] * C : item[u] * 2 * C;
    if (!turns) at[u] = a.rd + (item[u] - a.turned) * 2 * C;
    then[u] = apart ? a.rd / 2 + at[u] : at[u] + C;
    if (head[u] < 0) continue;
    const HeadRows& r = head[u] < a.Hq ? a.q : head[u] < a.Hq + a.Hkv ? a.k : a.v;
    const int of = head[u] < a.Hq ? head[u] : head[u] < a.Hq + a.Hkv ? head[u] - a.Hq : head[u] - a.Hq - a.Hkv;
    const raw* p = static_cast<const raw*>(r.p) + t * r.token + of * r.head;
    x[u].load(p + at[u]);
    if (then[u] < a.D) y[u].load(p + then[u]);
  }

  // the token's place: behind the last sequence position 0 and no page
  long p = 0, page = -1;
  int slot = 0;
  if (a.Hkv) {
    const int b = a.batch.sequence(t);
    if (b < a.batch.B) {
      const int n = a.batch.new_rows(b), i = t - a.batch.first_row(b), length = a.batch.length(b);
      p = (long)a.batch.lengths[b] - n + i;
      if (p >= 0 && p < length) {
        page = a.batch.page_of(b, (int)p);
        slot = (int)p - (int)a.batch.page.div((uint32_t)p) * (int)a.batch.page.d;
      }
    }
  }
  if (a.positions)
    p = a.positions64 ? static_cast<const long*>(a.positions)[t] : (long)static_cast<const int*>(a.positions)[t];
  for (int i = lane; i < a.rd / 2; i += 64) {
    const int angle = (int)(((uint64_t)p * a.frequencies[i]) >> 32);  // a turn is 2^32
    float s, c;
    sincospif((float)angle * 0x1p-31f, &s, &c);
    cosine[wave][i] = c * a.turn;
    sine[wave][i] = s * a.turn;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (head[u] < 0) continue;
    if (head[u] < a.Hq + a.Hkv && item[u] < a.turned) {
      const float *c = &cosine[wave][item[u] * C], *s = &sine[wave][item[u] * C];
      if (!a.interleaved || C == 1) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
          float f = E::load(x[u].e[i]), g = E::load(y[u].e[i]);
          turn_pair(f, g, c[i], s[i]);
          x[u].e[i] = E::store(f);
          y[u].e[i] = E::store(g);
        }
      } else {
        auto turn = [&](raw& lo, raw& hi, int i) {
          float f = E::load(lo), g = E::load(hi);
          turn_pair(f, g, c[i], s[i]);
          lo = E::store(f);
          hi = E::store(g);
        };
#pragma unroll
        for (int i = 0; i < C / 2; ++i) turn(x[u].e[2 * i], x[u].e[2 * i + 1], i);
#pragma unroll
        for (int i = 0; i < C / 2; ++i) turn(y[u].e[2 * i], y[u].e[2 * i + 1], C / 2 + i);
      }
    }
    raw* o;
    if (head[u] < a.Hq) {
      o = static_cast<raw*>(a.q_out) + t * a.out_token + head[u] * a.out_head;
    } else {
      if (page < 0) continue;
      const bool key = head[u] < a.Hq + a.Hkv;
      const CacheSteps& st = key ? a.kc : a.vc;
      o = static_cast<raw*>(key ? a.k_cache : a.v_cache) + page * st.page + slot * st.slot +
          (head[u] - a.Hq - (key ? 0 : a.Hkv)) * st.head;
    }
    x[u].store(o + at[u]);
    if (then[u] < a.D) y[u].store(o + then[u]);
  }
}

template <typename E, int C, int U>
int launch_units(RotateArgs a, hipStream_t st) {
  const int items = a.rd / (2 * C) + (a.D - a.rd + 2 * C - 1) / (2 * C);
  a.turned = a.rd / (2 * C);
  a.items = FastDiv(items);
  a.per_unit = std::max(1, 64 * U / items);
  const int groups = host_ceil_div(a.heads, a.per_unit);
  a.groups = FastDiv(groups);
  const long units = (long)a.batch.T * groups;
  if (units > 0x7ffffff0l) return QMOE_EINVAL;
  a.units = (int)units;
  const unsigned blocks = host_ceil_div(units, 4);
  hipLaunchKernelGGL((rotate_kernel<E, C, U>), dim3(std::min(blocks, GRID_X), host_ceil_div(blocks, GRID_X)), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

template <typename E, int C>
int launch_chunks(const RotateArgs& a, hipStream_t st) {
  // a unit holds at least one whole head
  const int items = a.rd / (2 * C) + (a.D - a.rd + 2 * C - 1) / (2 * C);
  if (items > 256) return launch_units<E, C, 8>(a, st);
  if (items > 64) return launch_units<E, C, 4>(a, st);
  // Two of 64 where many waves look their tokens' places up (1, 2, 3, 4 of 64, us: 2246 tokens of 32 + 16 heads
  // of 128 15.3, 14.2, 14.0, 14.5; 64 of 32 + 8 4.6, 4.9, 5.7, 6.2; without places, 8192 of 16 heads
  // of 256 22.4, 23.4, 23.6, 26.2).
  if (a.Hkv && (long)a.batch.T * a.heads * items > 64 * 8192) return launch_units<E, C, 2>(a, st);
  return launch_units<E, C, 1>(a, st);
}

template <typename E>
int launch(const RotateArgs& a, hipStream_t st) {
  constexpr int C = 16 / sizeof(typename E::raw);
  // Where a half of what turns is no whole pieces of 16 bytes, element by element: 8192 tokens of 32 heads of 96, 24
  // turned, 72.8 us (1.4 TB/s), 96 turned 20.1 (5.0).
  if (a.rd % (2 * C) == 0 && a.D % C == 0) return launch_chunks<E, C>(a, st);
  return launch_chunks<E, 1>(a, st);
}

int dispatch(const RotateArgs& a, int type, hipStream_t st) {
  if (type == QMOE_BF16) return launch<ElemBF16>(a, st);
  if (type == QMOE_F16) return launch<ElemF16>(a, st);
  if (type == QMOE_F32) return launch<ElemF32>(a, st);
  return QMOE_EINVAL;
}

bool bad_heads(int D, int rd, int interleaved, float turn) {
  return D < 1 || D > D_MAX || rd < 0 || rd > D || rd % 2 || (interleaved != 0 && interleaved != 1) ||
         !(turn - turn == 0.f);
}

}  // namespace

extern "C" {

int qmoe_rotate(const void* x, long x_token, long x_head, void* y, long y_token, long y_head, int type,
                const void* positions, int positions64, const void* frequencies, int rd, int interleaved, float turn,
                int T, int heads, int D, void* stream) {
  if (T < 0 || heads < 0 || !known_type(type) || bad_heads(D, rd, interleaved, turn)) return QMOE_EINVAL;
  if (T == 0 || heads == 0) return QMOE_OK;
  if (!x || !y || !positions || (rd && !frequencies)) return QMOE_EINVAL;
  RotateArgs a = {};
  a.q = {x, x_token, x_head}, a.q_out = y, a.out_token = y_token, a.out_head = y_head;
  a.batch.T = T;
  a.frequencies = static_cast<const uint64_t*>(frequencies), a.positions = positions, a.positions64 = positions64;
  a.interleaved = interleaved, a.Hq = a.heads = heads, a.D = D, a.rd = rd, a.turn = turn;
  return dispatch(a, type, (hipStream_t)stream);
}

int qmoe_append_kv(const void* k, long k_token, long k_head, const void* v, long v_token, long v_head, const void* q,
                   long q_token, long q_head, void* q_out, int type, void* k_cache, long k_page, long k_slot,
                   long k_cache_head, void* v_cache, long v_page, long v_slot, long v_cache_head, const void* table,
                   long table_ld, int table_width, const void* lengths, const void* starts, const void* positions,
                   int positions64, const void* frequencies, int rd, int interleaved, float turn, int T, int B, int Hq,
                   int Hkv, int D, int page, long n_pages, void* stream) {
  if (T < 0 || B < 0 || Hq < 0 || Hkv < 1 || !known_type(type) || bad_heads(D, rd, interleaved, turn))
    return QMOE_EINVAL;
  if (page < 1 || page > 1 << 30 || n_pages < 0 || table_width < 0 || table_ld < 0 || (!starts && T != B))
    return QMOE_EINVAL;
  if ((q == nullptr) != (q_out == nullptr) || (Hq > 0) != (q != nullptr)) return QMOE_EINVAL;
  if ((long)Hq + 2l * Hkv > 1 << 20 || (long)table_width * page > TOKENS_MAX) return QMOE_EINVAL;
  if (T == 0) return QMOE_OK;
  if (!k || !v || (rd && !frequencies) || missing(k_cache, v_cache, n_pages, table, table_width, lengths, B)) return QMOE_EINVAL;
  RotateArgs a = {};
  a.q = {q, q_token, q_head}, a.k = {k, k_token, k_head}, a.v = {v, v_token, v_head};
  a.q_out = q_out, a.out_token = (long)Hq * D, a.out_head = D;
  a.k_cache = k_cache, a.v_cache = v_cache;
  a.kc = {k_page, k_slot, k_cache_head}, a.vc = {v_page, v_slot, v_cache_head};
  a.batch.table = static_cast<const int*>(table), a.batch.lengths = static_cast<const int*>(lengths);
  a.batch.starts = static_cast<const int*>(starts);
  a.batch.table_ld = table_ld, a.batch.n_pages = n_pages, a.batch.T = T, a.batch.B = B, a.batch.width = table_width;
  a.batch.page = FastDiv(page);
  a.frequencies = static_cast<const uint64_t*>(frequencies), a.positions = positions, a.positions64 = positions64;
  a.interleaved = interleaved, a.Hq = Hq, a.Hkv = Hkv, a.heads = Hq + 2 * Hkv, a.D = D, a.rd = rd, a.turn = turn;
  return dispatch(a, type, (hipStream_t)stream);
}

}  // extern "C"
