// Log probabilities of given tokens, entropy and top alternatives of rows of logits.
//
//   Z = sum_v e^l_v;  logprob(v) = l_v - ln Z;  entropy = -sum_v p_v ln p_v
//
// over the allowed v, from m = max l, S = sum e^(l - m), D = sum e^(l - m) (l - m) (base 2
// inside): logprob(v) = (l_v - m) - ln S, entropy = ln S - D / S. Sums in fp32.
//
// The logits are read once, 16 bytes per load; each lane keeps the running m, S and D of what it
// has read, taken to a new maximum once per step of 4 loads. The top alternatives are found in the
// same pass: a wave keeps as candidates only the logits that reach a bound which k logits of the
// row are known to reach, and the few that are left at the end are ranked by counting. Many rows
// are bound by HBM, with about ten vector operations per logit close behind (4096 x 131072 bf16:
// 182 us, 5.9 TB/s, top 8 189 us; 1024 x 65536 fp32, top 20: 52 us, 5.2 TB/s). Fewer rows than CUs are
// bound by a workgroup's own steps; the longest of them are split and joined by a second launch
// (1 x 131072, top 20: 9.2 us, none 4.5; 48 rows, top 8: 12.8, none 8.4, under a mask 15.3 and 10.6).
// An unfinished last step costs as much as a whole one (333 x 50003, top 5: 19.9 us, 1.2 ps per
// logit, 131072 of them 28.2 us, 0.65 ps; 4096 rows, none: 98 us, 0.48 ps, and 181 us, 0.34 ps). Times
// are those of graphs over several states.
#include "elem_types.h"

#include <algorithm>

namespace {

constexpr int TOP_MAX = 32;
constexpr int V_MAX = 1 << 30, M_MAX = 1 << 30;  // with a workgroup's stride on top they stay within an int
constexpr int JOIN_THREADS = 256;
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
// e^(l - m) is zero in fp32 below this distance (base 2); l - m is not taken lower in D,
// where an infinite distance would meet the zero.
constexpr float FAR = -152.f;

struct LogprobArgs {
  const void* logits;
  const int64_t* tokens;
  const uint8_t* allowed;
  float* logprobs;
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  long ld, lda;
  int T, V, m, top;
};

// Max, sum and weighted sum of a part of a row.
struct Part {
  float m, s, d;
};

// Base of the exponents: an empty part (m = -inf) takes 0, so its terms are e^-inf = 0.
QMOE_DEV float base_of(float m) { return m == -INFINITY ? 0.f : m; }

QMOE_DEV float wave_max_f32(float v) {
  v = fmaxf(v, QMOE_DPPF(v, 0xB1));
  v = fmaxf(v, QMOE_DPPF(v, 0x4E));
  v = fmaxf(v, QMOE_DPPF(v, 0x141));
  v = fmaxf(v, QMOE_DPPF(v, 0x140));
  const int i = __float_as_int(v);
  return fmaxf(fmaxf(__int_as_float(__builtin_amdgcn_readlane(i, 0)), __int_as_float(__builtin_amdgcn_readlane(i, 16))),
               fmaxf(__int_as_float(__builtin_amdgcn_readlane(i, 32)), __int_as_float(__builtin_amdgcn_readlane(i, 48))));
}

// p taken to the maximum m >= p.m
QMOE_DEV Part moved(Part p, float m) {
  const float shift = (p.m - base_of(m)) * LOG2E, c = __builtin_amdgcn_exp2f(shift);
  return {m, c * p.s, c * (p.d + fmaxf(shift, FAR) * p.s)};
}

// The parts of a wave's lanes as one, the same in every lane.
QMOE_DEV Part wave_join(Part p) {
  p = moved(p, wave_max_f32(p.m));
  return {p.m, wave_sum_f32(p.s), wave_sum_f32(p.d)};
}

// Distinct 64-bit selection keys: larger logit, then lower id (-0 counts as 0). 0: none.
QMOE_DEV uint64_t key_of(float l, int v) {
  const uint32_t b = __float_as_uint(l + 0.f);
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((uint64_t)o << 32) | (uint32_t)~v;
}
QMOE_DEV int key_id(uint64_t k) { return (int)~(uint32_t)k; }
QMOE_DEV float key_logit(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

// ---------------------------------------------------------------- one wave's stream

// Candidates for the top alternatives that a wave keeps between compactions.
constexpr int CAP = 256;
constexpr int KEPT = CAP / 64;

// Low bits of a logit's order key that its type leaves alike for all values of one sign.
template <typename E>
constexpr int KEY_SHIFT = 0;
template <>
constexpr int KEY_SHIFT<ElemBF16> = 16;
template <>
constexpr int KEY_SHIFT<ElemF16> = 13;

QMOE_DEV uint32_t order_of(float l) { return (uint32_t)(key_of(l, 0) >> 32); }
QMOE_DEV float order_logit(uint32_t o) { return key_logit((uint64_t)o << 32); }

// The least float above a value below infinity.
QMOE_DEV float just_above(float v) {
  const int b = __float_as_int(v + 0.f);
  return __int_as_float(b >= 0 ? b + 1 : b - 1);
}

QMOE_DEV int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// The k-th largest of one value per lane, bit by bit from the top.
template <int BITS>
QMOE_DEV uint32_t wave_kth(uint32_t v, int k) {
  uint32_t r = 0;
#pragma unroll
  for (int b = BITS - 1; b >= 0; --b) {
    const uint32_t c = r | (1u << b);
    if (__popcll(__ballot(v >= c)) >= k) r = c;
  }
  return r;
}

// The logit of the k-th largest of one order key per lane.
template <typename E>
QMOE_DEV float wave_kth_logit(uint32_t order, int k) {
  constexpr int SH = KEY_SHIFT<E>;
  uint32_t o = wave_kth<32 - SH>(order >> SH, k) << SH;
  if (!(o & 0x80000000u)) o |= (1u << SH) - 1u;  // a negative value's low zeros are ones in its key
  return order_logit(o);
}

// A key that the k best of a wave's distinct keys, N per lane, reach and no other does (the
// bits are tried from the top until exactly k are left); 0 where there are fewer than k.
template <int N>
QMOE_DEV uint64_t wave_kth_key(const uint64_t (&key)[N], int k) {
  uint64_t kth = 0;
#pragma unroll 1
  for (int b = 63; b >= 0; --b) {
    const uint64_t c = kth | (1ull << b);
    int count = 0;
#pragma unroll
    for (int q = 0; q < N; ++q) count += __popcll(__ballot(key[q] >= c));
    if (count < k) continue;
    kth = c;
    if (count == k) break;
  }
  return kth;
}

// Keeps the k best of a wave's n candidates (n >= k). Returns a bound that their logits reach
// (the logit of no key, even NaN, where the bits end early: fmaxf with it is still a bound).
QMOE_DEV float compact(uint64_t* cand, int n, int k) {
  const int lane = threadIdx.x & 63;
  uint64_t key[KEPT];
#pragma unroll
  for (int q = 0; q < KEPT; ++q) key[q] = q * 64 + lane < n ? cand[q * 64 + lane] : 0;
  const uint64_t kth = wave_kth_key(key, k);
  int at = 0;
#pragma unroll
  for (int q = 0; q < KEPT; ++q) {
    const bool keep = key[q] && key[q] >= kth;
    const uint64_t mask = __ballot(keep);
    if (keep) cand[at + lanes_below(mask)] = key[q];
    at += __popcll(mask);
  }
  return key_logit(kth);
}

// The order key of the largest logit that the same lane of all waves has seen.
struct Tops {
  uint32_t v[64];
  QMOE_DEV void clear() {
    if (threadIdx.x < 64) v[threadIdx.x] = 0;
  }
  // Brings this lane's largest logit in and returns the key of the largest of all.
  QMOE_DEV uint32_t raise(float mine) {
    const uint32_t o = order_of(mine);
    return max(o, __hip_atomic_fetch_max(&v[threadIdx.x & 63], o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
  }
};

// A wave's running state: per lane the softmax sums and the largest logit of what it has read,
// per wave the candidates for the top k and two bounds that a logit has to pass to become one:
// - tau: k logits of this wave, at lower ids than what follows, are >= tau: only above it;
// - floor: k logits of the workgroup, at any ids, are >= floor: from it on.
// floor is the k-th largest of the 64 maxima over the same lane of all waves, which a wave looks
// up whenever it sees a logit above its bounds; what other waves bring in later only makes the
// bound weaker than it could be.
template <typename E, bool MASK, bool TOP>
struct Stream {
  bool infinite = MASK;
  Part p = {-INFINITY, 0.f, 0.f};
  float top = -INFINITY, tau = -INFINITY, floor = -INFINITY;
  int count = 0;

  // Adds the J pieces of P logits x.get(j, i), their sums first, so that the terms of a long row
  // are added in two levels. An infinite distance to the maximum would make D NaN (0 * inf): so
  // long as none is met, nothing is done about it; from then on distances are taken no lower than
  // FAR. A row's places past its end are such distances: waves that hold some in its last step do
  // that step twice.
  template <int P, int J, typename X>
  QMOE_DEV void add(X& x, float most) {
    p = moved(p, fmaxf(p.m, most));
    const float z = base_of(p.m);
    if (!infinite) {
      float s = 0.f, d = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float l = (x.get(j, i) - z) * LOG2E, e = __builtin_amdgcn_exp2f(l);
          s += e;
          d += e * l;
        }
        __builtin_amdgcn_sched_barrier(0);  // a piece at a time: few registers, more waves
      }
      infinite = __any(d != d);
      if (!infinite) {
        p.s += s, p.d += d;
        return;
      }
    }
    x.pin();
    float s = 0.f, d = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float l = (x.get(j, i) - z) * LOG2E, e = __builtin_amdgcn_exp2f(l);
        s += e;
        d += e * fmaxf(l, FAR);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    p.s += s, p.d += d;
  }

  // The same pieces' logits as candidates, piece j from id first + j * stride on. logit(id)
  // reads one of them from memory.
  template <int P, int J, typename X, typename F>
  QMOE_DEV void offer(X& x, const float (&piece_most)[J], float most, int first, int stride, Tops* tops, uint64_t* cand,
                      int k, F logit) {
    if (!__any(most > tau && most >= floor)) return;
    x.pin();
    top = fmaxf(top, most);
    floor = fmaxf(floor, wave_kth_logit<E>(tops->raise(top), k));
    // enough lanes of this wave reach the floor: what follows has to exceed it
    float next_tau = __popcll(__ballot(top >= floor)) >= k ? floor : tau;
    const float least = floor > tau ? floor : just_above(tau);
    int n = count;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (!__any(piece_most[j] >= least)) continue;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float l = x.get(j, i);
        const bool in = l >= least;
        const uint64_t mask = __ballot(in);
        if (mask == 0) continue;
        const int at = n + lanes_below(mask);
        if (in && at < CAP) cand[at] = key_of(l, first + j * stride + i);
        n += __popcll(mask);
      }
    }
    if (n > CAP) {
      // Too many at once (equal or ascending logits): once more, from the k-th best of the lanes'
      // best keys on, which tell equal logits apart; keeping the k best if it fills all the same.
      uint64_t best[1] = {0};
#pragma unroll 1
      for (int e = 0; e < J * P; ++e) {
        const int id = first + e / P * stride + e % P;
        const float l = logit(id);
        if (l >= least) best[0] = max(best[0], key_of(l, id));
      }
      const uint64_t from = wave_kth_key(best, k);
      n = count;
#pragma unroll 1
      for (int e = 0; e < J * P; ++e) {
        const int id = first + e / P * stride + e % P;
        const float l = logit(id);
        const uint64_t key = key_of(l, id);
        bool in = l >= least && key >= from;
        uint64_t mask = __ballot(in);
        if (n + __popcll(mask) > CAP) {
          const float kth = compact(cand, n, k);
          floor = fmaxf(floor, kth);
          next_tau = fmaxf(next_tau, kth);  // for what follows these logits, whose ids are in no order
          n = k;
          in = in && l >= floor;
          mask = __ballot(in);
        }
        if (in) cand[n + lanes_below(mask)] = key;
        n += __popcll(mask);
      }
    }
    count = n;
    tau = next_tau;
  }
};

// ---------------------------------------------------------------- a row's results

QMOE_DEV void emit_top(const LogprobArgs& a, int t, int rank, uint64_t key, Part p, float log_s, bool undefined) {
  const bool none = undefined || key == 0;
  a.top_ids[(long)t * a.top + rank] = none ? -1 : key_id(key);
  a.top_logprobs[(long)t * a.top + rank] = undefined ? NAN : key == 0 ? -INFINITY : (key_logit(key) - p.m) - log_s;
}

// A given token and its logit (-inf where it is not allowed), read before the row is.
struct Given {
  int64_t token;
  float logit;
};
template <typename E>
QMOE_DEV Given load_given(const LogprobArgs& a, int t, int j) {
  Given g = {-1, -INFINITY};
  if (j >= a.m) return g;
  g.token = a.tokens[(long)t * a.m + j];
  if (g.token >= 0 && g.token < a.V && (!a.allowed || a.allowed[(long)t * a.lda + g.token]))
    g.logit = E::load(static_cast<const typename E::raw*>(a.logits)[(long)t * a.ld + g.token]);
  return g;
}

template <typename E, int THREADS>
QMOE_DEV void emit_row(const LogprobArgs& a, int t, Given g, Part p, float log_s, bool undefined) {
  if (threadIdx.x == 0) a.entropy[t] = p.s == 0.f ? 0.f : log_s - LN2 * p.d / p.s;
  for (int j = threadIdx.x; j < a.m; j += THREADS) {
    if (j >= THREADS) g = load_given<E>(a, t, j);
    float r = 0.f;
    if (g.token >= a.V || (g.token >= 0 && undefined)) r = NAN;
    else if (g.token >= 0) r = g.logit == -INFINITY ? g.logit : (g.logit - p.m) - log_s;
    a.logprobs[(long)t * a.m + j] = r;
  }
}

// Ranks n candidates (distinct keys) by counting the greater ones, the whole workgroup;
// out(rank, key) for the first k ranks, key 0 where there are fewer.
template <int THREADS, typename F>
QMOE_DEV void rank_top(const uint64_t* list, int n, int k, F out) {
  for (int c = threadIdx.x; c < n; c += THREADS) {
    const uint64_t mine = list[c];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) rank += list[i] > mine;
    if (rank < k) out(rank, mine);
  }
  if ((int)threadIdx.x >= n && (int)threadIdx.x < k) out(threadIdx.x, 0);
}

template <typename E>
constexpr int PIECE = 16 / sizeof(typename E::raw);

// -inf in a word of the type's values.
template <typename E>
constexpr uint32_t MINUS_INF = 0xff80ff80u;
template <>
constexpr uint32_t MINUS_INF<ElemF16> = 0xfc00fc00u;
template <>
constexpr uint32_t MINUS_INF<ElemF32> = 0xff800000u;

// A thread's next PIECES pieces of a row, as loaded; pieces from `end` on and places that the mask
// takes out hold -inf.
template <typename E, bool MASK, int PIECES, int THREADS>
struct Pieces {
  static constexpr int N = PIECE<E>;
  RawVec<N, sizeof(typename E::raw)> v[PIECES];
  QMOE_DEV void load(const typename E::raw* x, const uint8_t* ok, int piece, int end) {
    uint32_t allow[PIECES][N / 4];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const long c = piece + j * THREADS;
#pragma unroll
      for (int i = 0; i < v[j].WORDS; ++i) v[j].w[i] = MINUS_INF<E>;
#pragma unroll
      for (int i = 0; i < N / 4; ++i) allow[j][i] = 0;
      if (c < end) {
        v[j].load(x + c * N);
        if constexpr (MASK) {
#pragma unroll
          for (int i = 0; i < N / 4; ++i) __builtin_memcpy(&allow[j][i], ok + c * N + 4 * i, 4);
        }
      }
    }
    if constexpr (MASK) {
#pragma unroll
      for (int j = 0; j < PIECES; ++j)
#pragma unroll
        for (int i = 0; i < N / 4; ++i) take_out(v[j].w + i * v[j].WORDS / (N / 4), allow[j][i]);
    }
  }
  // -inf for those of 4 logits whose byte is 0, two 16-bit values at a time.
  QMOE_DEV static void take_out(uint32_t* w, uint32_t allow) {
    if constexpr (sizeof(typename E::raw) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (allow >> (8 * i)) & 0xffu ? w[i] : MINUS_INF<E>;
    } else {
      const uint32_t one = ((((allow & 0x7f7f7f7fu) + 0x7f7f7f7fu) | allow) >> 7) & 0x01010101u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t keep = __umul24(__builtin_amdgcn_perm(0u, one, i ? 0x0c030c02u : 0x0c010c00u), 0xffffu);
        w[i] = (w[i] & keep) | (MINUS_INF<E> & ~keep);
      }
    }
  }
  // Unpacked again by what follows, not kept as 32-bit values.
  QMOE_DEV void pin() {
#pragma unroll
    for (int j = 0; j < PIECES; ++j)
#pragma unroll
      for (int i = 0; i < v[j].WORDS; ++i) asm volatile("" : "+v"(v[j].w[i]));
  }
  QMOE_DEV float get(int j, int i) const { return v[j].template get<E>(i); }
};

// A workgroup of WAVES waves takes one of `n_parts` parts of a row, in steps of PIECES pieces of 16
// bytes per thread; with one part it writes the row's results, with several its sums and its best
// candidates for join_kernel.
template <typename E, bool MASK, bool TOP, int PIECES, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void logprob_kernel(LogprobArgs a, int n_parts, int pieces_per_part, Part* parts,
                                                             uint64_t* keys) {
  constexpr int N = PIECE<E>, THREADS = 64 * WAVES;
  __shared__ uint64_t cand[TOP ? WAVES : 1][TOP ? CAP : 1], list[TOP ? WAVES * CAP : 1];
  __shared__ Part wave_part[WAVES];
  __shared__ Tops tops;
  __shared__ int listed;
  const int tid = threadIdx.x, wave = tid >> 6;
  if constexpr (TOP) {
    tops.clear();
    __syncthreads();
  }
  for (long unit = blockIdx.x; unit < (long)a.T * n_parts; unit += gridDim.x) {
    const int t = (int)(unit / n_parts), part = (int)(unit % n_parts);
    const auto* x = static_cast<const typename E::raw*>(a.logits) + (long)t * a.ld;
    const uint8_t* ok = MASK ? a.allowed + (long)t * a.lda : nullptr;
    const int pieces = a.V / N, begin = part * pieces_per_part, end = min(pieces, begin + pieces_per_part);
    const Given given = n_parts == 1 ? load_given<E>(a, t, tid) : Given{-1, 0.f};
    Stream<E, MASK, TOP> st;
    auto logit = [&](int v, int stop) { return v < stop && (!MASK || ok[v]) ? E::load(x[v]) : -INFINITY; };
    for (int q = begin; q < end; q += THREADS * PIECES) {
      Pieces<E, MASK, PIECES, THREADS> now;
      now.load(x, ok, q + tid, end);
      float most = -INFINITY, piece_most[PIECES];
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        piece_most[j] = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i) piece_most[j] = fmaxf(piece_most[j], now.get(j, i));
        most = fmaxf(most, piece_most[j]);
      }
      now.pin();
      st.template add<N, PIECES>(now, most);
      if constexpr (TOP)
        st.template offer<N, PIECES>(now, piece_most, most, (q + tid) * N, THREADS * N, &tops, cand[wave], a.top,
                                     [&](int id) { return logit(id, end * N); });
    }
    if (part == n_parts - 1 && pieces * N < a.V) {  // the row's end, less than a piece
      const int v = pieces * N + tid;
      struct {
        float l;
        QMOE_DEV float get(int, int) const { return l; }
        QMOE_DEV void pin() {}
      } last = {logit(v, a.V)};
      const float most[1] = {last.l};
      st.template add<1, 1>(last, last.l);
      if constexpr (TOP)
        st.template offer<1, 1>(last, most, last.l, v, 0, &tops, cand[wave], a.top,
                                [&](int id) { return logit(id, a.V); });
    }
    Part p = wave_join(st.p);
    if ((tid & 63) == 0) wave_part[wave] = p;
    if (tid == 0) listed = 0;
    __syncthreads();
    p = wave_join((tid & 63) < WAVES ? wave_part[tid & 63] : Part{-INFINITY, 0.f, 0.f});
    const bool undefined = !(p.s >= 0.f);  // a NaN or +inf at an allowed place
    const float log_s = logf(p.s);
    if constexpr (TOP) {
      const float floor = wave_kth_logit<E>(tops.raise(st.top), a.top);
      int above = 0;
      for (int i = 0; i < st.count; i += 64) {
        const int at = i + (tid & 63);
        above += __popcll(__ballot(at < st.count && key_logit(cand[wave][min(at, CAP - 1)]) >= floor));
      }
      if (above > 2 * TOP_MAX) {  // ranking many equal logits would take long
        compact(cand[wave], st.count, a.top);
        st.count = a.top;
      }
      for (int i = tid & 63; i < st.count; i += 64) {
        const uint64_t key = cand[wave][i];
        if (key_logit(key) >= floor) list[atomicAdd(&listed, 1)] = key;
      }
      __syncthreads();
      tops.clear();  // for the next row
      if (n_parts == 1)
        rank_top<THREADS>(list, listed, a.top, [&](int r, uint64_t k) { emit_top(a, t, r, k, p, log_s, undefined); });
      else
        rank_top<THREADS>(list, listed, a.top, [&](int r, uint64_t k) { keys[unit * a.top + r] = k; });
    }
    if (n_parts == 1) emit_row<E, THREADS>(a, t, given, p, log_s, undefined);
    else if (tid == 0) parts[unit] = p;
    __syncthreads();  // the next row reuses the LDS
  }
}

constexpr int MAX_PARTS = 64;  // one part per lane of the joining wave

// Joins the parts of a row: their sums and their ordered best candidates.
template <typename E, bool TOP>
__global__ __launch_bounds__(JOIN_THREADS) void join_kernel(LogprobArgs a, int n_parts, const Part* parts,
                                                            const uint64_t* keys) {
  constexpr int THREADS = JOIN_THREADS;
  constexpr int EACH = MAX_PARTS * TOP_MAX / THREADS;
  __shared__ uint64_t list[TOP ? MAX_PARTS * TOP_MAX : 1];
  __shared__ int listed;
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const Given given = load_given<E>(a, t, tid);
  Part p = {-INFINITY, 0.f, 0.f};
  if (lane < n_parts) p = parts[(long)t * n_parts + lane];
  uint64_t key[TOP ? EACH : 1];
  if constexpr (TOP) {
    const uint64_t* mine = keys + (long)t * n_parts * a.top;
    // The parts' keys are in order, so where `lists` parts have an r-th key of at least a floor
    // and r * lists >= k, k keys reach it.
    const int r = (a.top + n_parts - 1) / n_parts, lists = (a.top + r - 1) / r;
    const uint64_t rth = lane < n_parts ? mine[lane * a.top + r - 1] : 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) key[i] = i * THREADS + tid < n_parts * a.top ? mine[i * THREADS + tid] : 0;
    if (tid == 0) listed = 0;
    constexpr int SH = KEY_SHIFT<E>;
    uint64_t floor = (uint64_t)(wave_kth<32 - SH>((uint32_t)(rth >> 32) >> SH, lists) << SH) << 32;
    int above = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) above += __popcll(__ballot(key[i] && key[i] >= floor));
    // many equal or ascending logits: ranking all of them would take long
    if (above > 2 * TOP_MAX) floor = max(floor, wave_kth_key(key, a.top));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (key[i] && key[i] >= floor) list[atomicAdd(&listed, 1)] = key[i];
    __syncthreads();
  }
  p = wave_join(p);
  const bool undefined = !(p.s >= 0.f);
  const float log_s = logf(p.s);
  if constexpr (TOP) {
    rank_top<JOIN_THREADS>(list, listed, a.top, [&](int r, uint64_t k) { emit_top(a, t, r, k, p, log_s, undefined); });
  }
  emit_row<E, JOIN_THREADS>(a, t, given, p, log_s, undefined);
}

// How a call's rows go over workgroups.
struct Plan {
  int parts;   // of a row; more than one are joined by a second launch
  int pieces;  // of 16 bytes per part
  int waves;   // per workgroup
};

// Whole rows wherever they fill the chip or are short, which also saves the second launch;
// otherwise parts of whole steps of 4 pieces per thread (or one step of 2 or 1), up to 1024
// workgroups of 4 waves. V in bf16, top 8, split and whole on 16 waves: 1 row of 65536 8.4 and 9.7
// us, of 131072 8.5 and 14.3; 64 rows 12.0 and 10.8, 13.9 and 15.8; 128 rows 14.1 and 11.2, 18.4 and
// 17.3; 192 rows of 131072 21.7 and 17.7. Parts of 131072, top 20: 1, 2, 4, 8, 16, 32, 64 of them
// take 26.9, 20.9, 15.9, 12.5, 10.7, 9.9 and 9.4 us for 1 row, 31.2, 24.5, 18.3, 15.7, 14.4, 14.9 and
// 20.2 for 48.
// Waves for whole rows: 16 with up to a row per CU and enough in it, 8 with up to two rows per CU or
// short rows, 4 for more rows, where the waves of several rows hide each other's latency. Top 8, 4, 8
// and 16 waves: 64 x 32768 11.6, 8.9 and 8.1; 64 x 8192 6.2, 5.7 and 6.4; 333 x 32768 14.7, 12.3 and
// 15.6; 333 x 8192 7.5, 7.6 and 11.6; 1024 x 32768 20.5, 23.1 and 30.4. Without top alternatives, whose
// candidates each wave pays for, 8 waves win for many rows as well (2048 x 65536 55.7 and 52.6;
// 4096 x 131072 194 and 184; but 1024 x 131072 52.8 and 54.8).
Plan plan_for(int T, int V, int type, int top) {
  const int pieces = V / (type == QMOE_F32 ? 4 : 8);
  if (pieces <= 4096 || T >= 160 || pieces <= 128 * T) {
    int waves = 4;
    if (T <= 256) waves = pieces >= 4096 ? 16 : 8;
    else if (T <= 512) waves = pieces >= 2048 ? 8 : 4;
    else if (T > 1024 && !top) waves = pieces >= 4096 ? 8 : 4;
    return {1, std::max(pieces, 1), waves};
  }
  constexpr int STEP = 256;
  const int want = std::min(1024 / T, MAX_PARTS);
  for (int per = STEP; per < 4 * STEP; per *= 2)
    if (host_ceil_div(pieces, per) <= want) return {host_ceil_div(pieces, per), per, 4};
  const int per = 4 * STEP * host_ceil_div(host_ceil_div(pieces, 4 * STEP), want);
  return {host_ceil_div(pieces, per), per, 4};
}

size_t parts_bytes(int T, const Plan& p) { return ((size_t)T * p.parts * sizeof(Part) + 15) / 16 * 16; }

template <typename E, bool MASK, bool TOP, int STEP, int WAVES>
void launch_rows(const LogprobArgs& a, const Plan& p, Part* parts, uint64_t* keys, hipStream_t st) {
  const unsigned grid = (unsigned)std::min<long>((long)a.T * p.parts, 1l << 20);
  hipLaunchKernelGGL((logprob_kernel<E, MASK, TOP, STEP, WAVES>), dim3(grid), dim3(64 * WAVES), 0, st, a, p.parts, p.pieces,
                     parts, keys);
}

template <typename E, bool MASK, bool TOP>
int launch(const LogprobArgs& a, const Plan& p, void* ws, hipStream_t st) {
  Part* parts = static_cast<Part*>(ws);
  uint64_t* keys = p.parts > 1 ? reinterpret_cast<uint64_t*>(static_cast<char*>(ws) + parts_bytes(a.T, p)) : nullptr;
  const int each = host_ceil_div(p.pieces, 64 * p.waves);  // pieces per thread
  if (p.waves == 16) launch_rows<E, MASK, TOP, 4, 16>(a, p, parts, keys, st);
  else if (p.waves == 8 && each == 1) launch_rows<E, MASK, TOP, 1, 8>(a, p, parts, keys, st);
  else if (p.waves == 8 && each == 2) launch_rows<E, MASK, TOP, 2, 8>(a, p, parts, keys, st);
  else if (p.waves == 8) launch_rows<E, MASK, TOP, 4, 8>(a, p, parts, keys, st);
  else if (each == 1) launch_rows<E, MASK, TOP, 1, 4>(a, p, parts, keys, st);
  else if (each == 2) launch_rows<E, MASK, TOP, 2, 4>(a, p, parts, keys, st);
  else launch_rows<E, MASK, TOP, 4, 4>(a, p, parts, keys, st);
  if (p.parts > 1)
    hipLaunchKernelGGL((join_kernel<E, TOP>), dim3(a.T), dim3(JOIN_THREADS), 0, st, a, p.parts, parts, keys);
  return (int)hipGetLastError();
}

template <typename E>
int dispatch(const LogprobArgs& a, const Plan& p, void* ws, hipStream_t st) {
  if (a.allowed) return a.top ? launch<E, true, true>(a, p, ws, st) : launch<E, true, false>(a, p, ws, st);
  return a.top ? launch<E, false, true>(a, p, ws, st) : launch<E, false, false>(a, p, ws, st);
}

}  // namespace

extern "C" {

size_t qmoe_token_logprobs_workspace(int T, int V, int type, int top) {
  if (T < 1 || V < 1 || top < 0 || top > TOP_MAX || !known_type(type)) return 0;
  const Plan p = plan_for(T, V, type, top);
  return p.parts == 1 ? 0 : parts_bytes(T, p) + (size_t)T * p.parts * top * sizeof(uint64_t);
}

int qmoe_token_logprobs(const void* logits, long ld, int type, const void* tokens, int m, const void* allowed,
                        long ld_allowed, int T, int V, void* logprobs, void* entropy, int top, void* top_ids,
                        void* top_logprobs, void* workspace, size_t workspace_bytes, void* stream) {
  if (T < 0 || V < 1 || V > V_MAX || m < 0 || m > M_MAX || top < 0 || top > TOP_MAX || ld < 0 ||
      (allowed && ld_allowed < 0) || !known_type(type))
    return QMOE_EINVAL;
  if (T == 0) return QMOE_OK;
  if (!logits || !entropy || (m && (!tokens || !logprobs)) || (top && (!top_ids || !top_logprobs))) return QMOE_EINVAL;
  const size_t need = qmoe_token_logprobs_workspace(T, V, type, top);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return QMOE_EWORKSPACE;
  LogprobArgs a = {};
  a.logits = logits, a.ld = ld, a.tokens = (const int64_t*)tokens, a.m = m;
  a.allowed = (const uint8_t*)allowed, a.lda = ld_allowed, a.T = T, a.V = V;
  a.logprobs = (float*)logprobs, a.entropy = (float*)entropy;
  a.top = top, a.top_ids = (int64_t*)top_ids, a.top_logprobs = (float*)top_logprobs;
  const Plan p = plan_for(T, V, type, top);
  if (type == QMOE_BF16) return dispatch<ElemBF16>(a, p, workspace, (hipStream_t)stream);
  if (type == QMOE_F16) return dispatch<ElemF16>(a, p, workspace, (hipStream_t)stream);
  return dispatch<ElemF32>(a, p, workspace, (hipStream_t)stream);
}

}  // extern "C"
