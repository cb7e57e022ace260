// Attention of new tokens over the pages of their sequences.
//
// Row (t, h) at position p of its sequence sees the keys j with p - window < j <= p that lie on a
// page of the cache:  o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale * q.k_j,
// m = max_j s_j. Scores, sums and the output's sums in fp32, each output rounded once. A row that sees no key, or
// whose scores are all -inf, gives 0.
//
// The weights e^(s_j - m) are rounded to the tensors' type, as the matrix instructions take their operands (in two
// 16-bit parts each the second product would take twice as long), and summed after it, so that their sum is that of
// what multiplies v. Error of the outputs, relative to their norm, with these weights and with weights in
// fp32: bf16 0.0019 and 0.0017 (1 token after 4096), 0.0021 and 0.0016 (8192 tokens), 0.0022 and 0.0016 (4 after 131072,
// heads of 256); fp16 0.00022 and 0.00021, under a window 0.00027 and 0.00021.
//
// One pass over the keys with a running maximum and sum. The rows that share a key head (a sequence's
// tokens times the query heads of the group) are one matrix; a wave holds 32 of them. It takes
// S^T = K Q^T and O^T += V^T P^T on 32 x 32 x 16 MFMAs: a lane then holds scores of one row only (lane & 31),
// so that maximum and sum are sums over its own registers and one exchange with lane ^ 32, and the
// weights lie in registers just as the second product reads them, once the keys of 16 are taken in the
// order 4 half + (i & 3) + 8 (i >> 2). V's columns for it come out of LDS with transposing reads.
//
// Two ways to cut the work, in one launch:
//  * sequences with more than 32 rows: 128 rows to a workgroup, which its four waves share out, and 64 keys
//    at a time in LDS for all of them; where such tiles are few, their keys are cut into pieces;
//  * sequences with up to 32 rows (single tokens): the waves of a workgroup hold the same rows and
//    share out the keys, 32 each at a time. All keys of all such sequences and heads make one list
//    of tiles of 128, of which every workgroup takes an equal share, however the lengths differ.
// What lies in pieces or crosses shares is joined by a second launch.
#include "attention_layout.h"
#include "paged.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace {

typedef float f32x16_v __attribute__((ext_vector_type(16)));
typedef float f32x4_v __attribute__((ext_vector_type(4)));
typedef short s16x4_v __attribute__((ext_vector_type(4)));
typedef short s16x8_v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;

constexpr int ROWS = 128;      // rows of a workgroup, many-rows form
constexpr int FEW = 32;        // rows up to which a sequence takes the few-rows form
constexpr int FEW_KEYS = 128;  // keys of a tile of that form
constexpr int FEW_BLOCKS_MAX = 768;  // workgroups of that form, and parts of a row
constexpr int D_MAX = 256, GROUP_MAX = 64;

struct AttentionArgs {
  const void *q, *k, *v;
  void* out;
  long q_token, q_head;
  CacheSteps kc, vc;
  Batch batch;
  int Hq, Hkv, D, window;
  FastDiv group, heads;
  float scale;      // |scale| * log2(e), above 0
  int negate;       // of a scale below 0
  int same_pages;   // 16 keys on 16 lie on one page
  int few;          // FEW, or 0: all sequences take the many-rows form
  int few_blocks, few_from, few_rows, many_tiles, pieces, slots;
  int join_few, join_many;  // workgroups that share out the rows of a head of few rows, of a tile
  float *few_part, *many_part;  // partial sums: rows of D, then pairs (maximum, sum)
};

// Maxima and sums behind the partial sums' rows.
QMOE_DEV float2* few_tops(const AttentionArgs& a) {
  return reinterpret_cast<float2*>(a.few_part + 2l * a.few_blocks * a.few_rows * a.D);
}
QMOE_DEV float2* many_tops(const AttentionArgs& a) {
  return reinterpret_cast<float2*>(a.many_part + 2l * (2 * a.slots + 1) * ROWS * a.D);
}

// Inclusive sums over a wave's lanes.
QMOE_DEV int prefix_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15: to rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31: to rows 2 and 3
  return v;
}
QMOE_DEV int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
// A byte offset of lane `src` (wave-uniform) as a scalar.
QMOE_DEV long read_lane(long v, int src) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)v, src), hi = __builtin_amdgcn_readlane((int)(v >> 32), src);
  return (long)(((uint64_t)hi << 32) | lo);
}
// What lanes of a wave write to LDS, for the others of it.
QMOE_DEV void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <typename E>
struct Mma;
template <>
struct Mma<ElemBF16> {
  using frag = bf16x8_v;
  QMOE_DEV static f32x16_v mma(s16x8_v a, s16x8_v b, f32x16_v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
  QMOE_DEV static uint32_t pack(float lo, float hi) { return pk_bf16(lo, hi); }
  // sum + both elements, in fp32
  QMOE_DEV static float add_pair(uint32_t v, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_v, v), __builtin_bit_cast(bf16x2_v, 0x3f803f80u), sum, false);
  }
  static constexpr uint32_t EXPONENT = 0x7f807f80u, ONE = 0x00800080u;
};
template <>
struct Mma<ElemF16> {
  using frag = f16x8_v;
  QMOE_DEV static f32x16_v mma(s16x8_v a, s16x8_v b, f32x16_v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
  QMOE_DEV static uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_v){lo, hi}, f16x2_v));
  }
  QMOE_DEV static float add_pair(uint32_t v, float sum) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_v, v), __builtin_bit_cast(f16x2_v, 0x3c003c00u), sum, false);
  }
  static constexpr uint32_t EXPONENT = 0x7c007c00u, ONE = 0x04000400u;
};

// Maximum and sum with lane ^ 32.
QMOE_DEV float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
QMOE_DEV float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A lane's row sees the keys [low, high], of those that are present in a tile.
struct Seen {
  int low, high;
};

// 32 rows of a wave against NJ blocks of 32 keys.
template <typename E, int NK, int NJ>
struct Rows {
  using L = Layout<NK>;
  f32x16_v o[NK];  // o[dt][r]: element 32 dt + 8 (r >> 2) + 4 half + (r & 3) of row lane & 31
  float m, l;      // a score that weights are relative to, in units of log2; sum of this half's weights

  QMOE_DEV void clear() {
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int dt = 0; dt < NK; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  }

  // Number in the tile of the key in register r of block j, in lanes of the first half; 4 more in the others.
  QMOE_DEV static constexpr int key_of(int j, int r) { return 32 * j + 8 * (r >> 2) + (r & 3); }

  // Scores s become weights p = 2^(scale s - m); returns their sum over this lane's keys. m is the maximum of the
  // keys of some tile and moves only where that sum exceeds 2^12: weights below that are held by fp32 and the 16-bit
  // types as well as those below 1, so most tiles need no maximum and leave the output's sums alone.
  QMOE_DEV float weigh(const f32x16_v (&s)[NJ], float scale, s16x8_v (&p)[2 * NJ]) const {
    const float base = m == -INFINITY ? 0.f : m;
    float sum[2] = {};
#pragma unroll
    for (int i = 0; i < 2 * NJ; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = 8 * (i & 1) + 2 * r;
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 2][at], scale, -base));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 2][at + 1], scale, -base));
        w[r] = Mma<E>::pack(x, y);
        sum[r & 1] = Mma<E>::add_pair(w[r], sum[r & 1]);
      }
      p[i] = __builtin_bit_cast(s16x8_v, (u32x4_v){w[0], w[1], w[2], w[3]});
    }
    return sum[0] + sum[1];
  }
  // Whether a row needs another m for weights of that sum (any, if it has none yet).
  QMOE_DEV bool moves(float sum) const { return __any(sum > (m == -INFINITY ? -1.f : 0x1p12f)); }
  // m becomes the maximum of these scores, where it is below; all weights before must be in o and l.
  QMOE_DEV void move(const f32x16_v (&s)[NJ], float scale) {
    float t = s[0][0];
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) t = fmaxf(t, s[j][r]);
    const float top = fmaxf(m, half_max(t) * scale), f = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
    m = top, l *= f;
#pragma unroll
    for (int dt = 0; dt < NK; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] *= f;
  }
  // weigh() with the maximum moved if need be; what comes before must be in o.
  QMOE_DEV void settle(const f32x16_v (&s)[NJ], float scale, s16x8_v (&p)[2 * NJ], float sum) {
    if (moves(sum)) {
      move(s, scale);
      sum = weigh(s, scale, p);
    }
    l += sum;
  }

  // o += V^T p, V's rows in LDS. A lane of a transposing read names 4 elements of a row: in groups of 16 lanes,
  // lane i row i >> 2 and elements 4 (i & 3) of 16; it gets element i of the four rows.
  QMOE_DEV void add(const unsigned char* v, const s16x8_v (&p)[2 * NJ]) {
    const int lane = threadIdx.x & 63, half = lane >> 5, row = 4 * half + ((lane >> 2) & 3);
    const int piece = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1), swizzle = L::v_swizzle(row);
    const unsigned char* base = v + row * L::STRIDE + 8 * (lane & 1);
#pragma unroll
    for (int i = 0; i < 2 * NJ; ++i)
#pragma unroll
      for (int dt = 0; dt < NK; ++dt) {
        const unsigned char* at = base + 16 * i * L::STRIDE + 16 * ((4 * dt + piece) ^ swizzle);
        typedef __attribute__((address_space(3))) s16x4_v lds_frag;
        const s16x4_v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_frag*)at);
        const s16x4_v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_frag*)(at + 8 * L::STRIDE));
        o[dt] = Mma<E>::mma(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7), p[i], o[dt]);
      }
  }

  // Scores of keys `first` and so on: those that the row does not see become -inf.
  QMOE_DEV static void mask(f32x16_v (&s)[NJ], Seen seen, uint64_t present, int first) {
    const int half = (threadIdx.x >> 5) & 1, from = first + 4 * half;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int low = seen.low - from - 32 * j, high = seen.high - from - 32 * j;
      uint32_t bits = (uint32_t)(present >> (32 * j)) >> (4 * half);
      bits = low > 31 || high < 0 ? 0 : bits & ~0u << max(low, 0) & ~0u >> (31 - min(high, 31));
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!((bits >> (key_of(j, r) & 31)) & 1)) s[j][r] = -INFINITY;
    }
  }

  // The infinite and NaN values of 32 keys, which were left out of their tile: o += p v where the row sees the key (a
  // bit of `there` each, the first one key `first`), p its weight, rounded as in whole tiles, so that a score of -inf
  // gives NaN here as there. k + ko and v + vo: the row of key `lane & 31`; q(ks): the second operand of K Q^T;
  // w: 4 KB of LDS that only this wave uses.
  template <bool FULL, typename Q>
  QMOE_DEV void add_unusual(const unsigned char* k, long ko, const unsigned char* v, long vo, uint32_t there, int first, Seen seen,
                            float scale, Q q, float* w, int D) {
    // (no registers for sums of the lane, offsets of elements or loads ahead: the loop before needs them)
    int lane = threadIdx.x & 63;
    if (!FULL) asm volatile("" : "+v"(lane));
    const int half = lane >> 5;
    int part = 16 * half, row_of = lane & 31;
    asm volatile("" : "+v"(part), "+v"(row_of));
    f32x16_v s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 2 * NK; ++ks) {
      const bool within = FULL || L::always(ks) || 16 * ks + 8 * half < D;
      u32x4_v f = *reinterpret_cast<const u32x4_v*>(k + ko + (within ? 32 * ks + part : 0));
      if (!within) f = (u32x4_v){0, 0, 0, 0};
      s = Mma<E>::mma(__builtin_bit_cast(s16x8_v, f), q(ks), s);
      __builtin_amdgcn_sched_barrier(0);
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale, -base));
      w[(key_of(0, r) + 4 * half) * 32 + row_of] = E::load((uint16_t)Mma<E>::pack(p, p));
    }
    wave_fence();
#pragma unroll 1
    for (int i = 0; i < 32; ++i) {
      const bool is = (there >> i) & 1, sees = is && first + i >= seen.low && first + i <= seen.high;
      const unsigned char* row = v + (is ? read_lane(vo, i) : 0);
      const float p = w[i * 32 + row_of];
      int last = D - 4;
      if (!FULL) asm volatile("" : "+s"(last));
#pragma unroll
      for (int dt = 0; dt < NK; ++dt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int d = 32 * dt + 8 * c + 4 * half;
          const s16x4_v x = *reinterpret_cast<const s16x4_v*>(row + 2 * (FULL ? d : min(d, last)));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = E::load((uint16_t)x[e]);
            if (sees && !(f - f == 0.f)) o[dt][4 * c + e] += p * f;
          }
        }
    }
    wave_fence();
  }
};

// Values of V that some rows of a tile see and others do not: a weight of 0 times an infinity or NaN would
// be NaN. So in tiles that not every row sees whole, such values become 0 (COUNT KB at v + `every` KB each,
// as this wave loaded them); the rows that see them get them after the loop. Returns whether there were any.
template <typename E, int COUNT>
QMOE_DEV bool clean(unsigned char* v, int every) {
  u32x4_v* at = reinterpret_cast<u32x4_v*>(v) + (threadIdx.x & 63);
  u32x4_v w[COUNT];
#pragma unroll
  for (int g = 0; g < COUNT; ++g) w[g] = at[g * every * 64];
  uint32_t any = 0;
#pragma unroll
  for (int g = 0; g < COUNT; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= (w[g][i] & Mma<E>::EXPONENT) + Mma<E>::ONE;
  if (!__any((any & 0x80008000u) != 0)) return false;
#pragma unroll 1
  for (int g = 0; g < COUNT; ++g) {
    u32x4_v x = at[g * every * 64];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = (x[i] & Mma<E>::EXPONENT) + Mma<E>::ONE;
      if (u & 0x8000u) x[i] &= 0xffff0000u;
      if (u & 0x80000000u) x[i] &= 0xffffu;
    }
    at[g * every * 64] = x;
  }
  return true;
}

// Elements at, at + 1, .. at + 7 of a row of q.
QMOE_DEV s16x8_v q_piece(const uint16_t* row, int at, int D, bool valid, int negate) {
  u32x4_v w = {0, 0, 0, 0};
  if (valid && at < D) {
    w = *reinterpret_cast<const u32x4_any*>(row + at);
    if (negate) w ^= 0x80008000u;
  }
  return __builtin_bit_cast(s16x8_v, w);
}

// Positions of a sequence's rows, as ints: what precedes its first new token, clamped.
QMOE_DEV int tokens_before(const Batch& batch, int b, int n) {
  return (int)max((long)batch.lengths[b] - n, -0x40000000l);
}

// COUNT runs of rows, one 16-byte piece per lane, straight to LDS: run g is rows src + g * EVERY of the
// tile, whose offsets the lanes hold, to `to` + 1 KB * g * EVERY / RPI. Lanes past a head's elements
// load its last piece again, as a load to LDS without some of its lanes takes several times as long (32 tokens
// after up to 16384, 8 heads of 80: 226 us, so 62): such values of V only reach sums that are not stored, those
// of K are made 0 where they are read, or not read. A row that is not there is skipped, or zeroed; the cache's first row in
// its place, for all such rows of all tiles, took longer (8 sequences of up to 500 after up to 30000 369 us, 412).
// `run`: 16 rows on 16 lie one step apart, so that an offset of each 16, as a scalar, does for all of them.
template <int NK, bool FULL, int COUNT, int EVERY, bool KEYS>
QMOE_DEV void load_rows(unsigned char* to, const unsigned char* base, long offset, uint64_t present, bool whole, bool run,
                        int src, uint32_t step, int D) {
  using L = Layout<NK>;
  const int lane = threadIdx.x & 63, row = lane / L::PIECES;
  auto piece_of = [&](int mine) { return L::template piece_of<FULL, KEYS>(lane, mine, D); };
  if (whole && run) {
#pragma unroll
    for (int g = 0; g < COUNT; ++g) {
      // (opaque, so that no sums of the base and a lane's offset are kept over the loop)
      const int from = src + g * EVERY;
      uint64_t p = reinterpret_cast<uint64_t>(base) + read_lane(offset, from & ~15) + (from & 15) * step;
      asm volatile("" : "+s"(p));
      const int piece = piece_of(from + row);
      __builtin_amdgcn_global_load_lds((global_void*)(p + (row * step + 16u * piece)),
                                       (lds_void*)(to + g * (1024 * EVERY / L::RPI)), 16, 0, 0);
    }
  } else {
#pragma unroll 1
    for (int g = 0; g < COUNT; ++g) {
      const int mine = src + g * EVERY + row, piece = piece_of(mine);
      unsigned char* at = to + g * (1024 * EVERY / L::RPI);
      const long from = __shfl(offset, mine);
      if ((present >> mine) & 1)
        __builtin_amdgcn_global_load_lds((global_void*)(base + from + 16 * piece), (lds_void*)at, 16, 0, 0);
      else if (!KEYS)
        *reinterpret_cast<u32x4_v*>(at + 16 * lane) = (u32x4_v){0, 0, 0, 0};
    }
  }
}

// Bytes of a cache's row of position `key` on page `entry` (0 for none).
QMOE_DEV long row_offset(const CacheSteps& c, const FastDiv& page, int entry, int key) {
  const uint32_t slot = key - page.div(key) * page.d;
  return entry < 0 ? 0 : (long)((uint64_t)(uint32_t)entry * (uint32_t)(2 * c.page) + slot * (uint32_t)(2 * c.slot));
}

// ---------------------------------------------------------------- sequences of many rows

// A tile of 128 rows of a sequence of many, or of the rows behind the last one (b = B, no keys).
struct ManyTile {
  int b, row0, rows, r0, before, begin, tiles;
};
// All such tiles, sequence after sequence.
struct ManyList {
  int rows, total;  // of sequence `lane`; tiles of all
  QMOE_DEV static int tiles_of(const AttentionArgs& a, int s, int rows) {
    return s < a.batch.B && rows <= a.few ? 0 : (rows + ROWS - 1) / ROWS;
  }
  QMOE_DEV static int rows_of(const AttentionArgs& a, int s) {
    return (s < a.batch.B ? a.batch.new_rows(s) : s == a.batch.B ? a.batch.T - a.batch.start(s) : 0) * (int)a.group.d;
  }
  QMOE_DEV ManyList(const AttentionArgs& a) {
    const int lane = threadIdx.x & 63;
    rows = rows_of(a, lane);
    int sum = tiles_of(a, lane, rows);
    for (int s = 64 + lane; s <= a.batch.B; s += 64) sum += tiles_of(a, s, rows_of(a, s));
    total = lane_of(prefix_sum(sum), 63);
  }
  // Tile `number` < total.
  QMOE_DEV ManyTile find(const AttentionArgs& a, int number) const {
    const int lane = threadIdx.x & 63;
    const Batch& batch = a.batch;
    ManyTile t = {};
    int first = 0;
    for (int i = 0; i <= batch.B; i += 64) {
      const int r = i ? rows_of(a, i + lane) : rows, mine = tiles_of(a, i + lane, r), upto = first + prefix_sum(mine);
      const uint64_t past = __ballot(upto > number);
      if (past) {
        const int at = __ffsll((unsigned long long)past) - 1;
        t.b = i + at, t.rows = lane_of(r, at), first = lane_of(upto - mine, at);
        break;
      }
      first = lane_of(upto, 63);
    }
    const bool is = t.b < batch.B;
    const int G = a.group.d, n = a.group.div(t.rows);
    t.row0 = batch.start(t.b), t.r0 = (number - first) * ROWS;
    t.before = is ? tokens_before(batch, t.b, n) : -0x40000000;
    const int first_pos = t.before + (int)a.group.div(t.r0), last_pos = t.before + (int)a.group.div(min(t.r0 + ROWS, t.rows) - 1);
    const int end = min(last_pos + 1, is ? batch.length(t.b) : 0);
    t.begin = a.window ? max(first_pos - a.window + 1, 0) & ~63 : 0;
    t.tiles = end > t.begin ? (end - t.begin + 63) / 64 : 0;
    return t;
  }
};

// Where tiles are few, long ones are cut into pieces. Tiles of a sequence count alike, with the most keys that one
// of them may see. Where all sequences' tiles are about as long, a piece is the part of all keys that one of the
// workgroups that run at once gets; else half of it, in tiles of more than two such pieces, so that long
// tiles do not outlast the rest. Shares and halves, us: 64 new tokens after 32768 70, 90 and after 65536 (heads
// of 256) 156, 187; 8 sequences of up to 500 after up to 30000 450, 393, heads of 192 1203, 939.
// In the list of all tiles' keys (sequence, tile, head), a piece that starts in stretch u of a piece's size is
// kept at 2 u, or 2 u + 1 if it is the first of its tile: a tile in pieces is longer than a stretch, so these
// differ.
// Tiles of up to that many times 64 keys are sooner done in one go than in pieces and a joining launch. us whole and
// in pieces: heads of 128, a prompt of 1024 (16) 34, 54, 64 tokens after 1024 (17) 32, 29, 256 after 2048 (36) 61, 39;
// heads of 256, whose steps take twice as long, a prompt of 2048 (saves 16 at most) 109, 118, 64 tokens after
// 1100 (19) 65, 45.
__host__ QMOE_DEV constexpr int whole_tiles(int D) { return D > 128 ? 16 : 24; }
struct Pieces {
  int size, start, whole;  // in units of 64 keys: a piece; this tile's start in the list; tiles up to that length are not cut
};
QMOE_DEV Pieces pieces_of(const AttentionArgs& a, const ManyTile& t, int h) {
  const int lane = threadIdx.x & 63, G = a.group.d;
  const Batch& batch = a.batch;
  int total = 0, count = 0, before = 0, of = 0;
  uint32_t most = 0;
  for (int i = 0; i < batch.B; i += 64) {
    int tiles = 0, keys = 0;
    if (i + lane < batch.B) {
      const int n = batch.new_rows(i + lane), rows = n * G;
      if (rows > a.few) {
        tiles = (rows + ROWS - 1) / ROWS;
        keys = min(tokens_before(batch, i + lane, n) + n, batch.length(i + lane));
        keys = (max(keys, 0) + 63) / 64;
        if (a.window) keys = min(keys, (a.window + ROWS / G + 64) / 64 + 1);
        keys = max(keys, 1);
      }
    }
    const int mine = tiles * keys * a.Hkv, upto = prefix_sum(mine);
    if (t.b >= i && t.b < i + 64) before = total + lane_of(upto - mine, t.b - i), of = lane_of(keys, t.b - i);
    total += lane_of(upto, 63);
    count += lane_of(prefix_sum(tiles * a.Hkv), 63);
    most = max(most, (uint32_t)lane_of((int)wave_max_u32_vec((uint32_t)keys), 0));
  }
  const bool alike = 4l * most * count <= 5l * total;
  const int stretches = alike ? a.slots : 2 * a.slots;
  const int size = max(8, (total + stretches - 1) / stretches);
  return {size, before + (t.r0 / ROWS * a.Hkv + h) * of, max(alike ? size : 2 * size, whole_tiles(a.D))};
}
QMOE_DEV int piece_count(const AttentionArgs& a, const Pieces& p, int tiles) {
  return tiles > p.whole ? min((tiles + p.size - 1) / p.size, a.pieces) : 1;
}
// (within the workspace also where sequences share rows against the rules, and their sums pass 32 bits)
QMOE_DEV long piece_at(const AttentionArgs& a, const Pieces& p, int piece) {
  const uint32_t stretch = ((uint32_t)p.start + (uint32_t)piece * (uint32_t)p.size) / (uint32_t)p.size;
  return 2l * min(stretch, 2u * a.slots) + (piece == 0);
}

// A workgroup: 128 rows against one piece of their keys, 64 at a time. K and V come to LDS by DMA, both
// halves of a double buffer, and serve four waves of 32 rows, so that a CU's two workgroups draw 128 KB of
// tiles for 256 rows' products; with heads of up to 128 two waves a SIMD hold q, the output's sums and the
// scores in 256 registers each. What bounds it is issue: of a step of 64 keys (heads of 128) a wave
// spends 4345 clocks, 1024 of them in its own 32 MFMAs, the rest in sharing the matrix pipe with the other
// wave of its SIMD (busy 38 %), in the weights (224 vector operations a tile; the vector pipe is busy 40 %)
// and in 450 at the wait and the barrier. 8192 tokens of 32 + 8 heads of 128, bf16: 584 us, 941 TFLOP/s, where a large
// product reaches 1235. Not faster there, us (in turn with what was there then): K loaded a tile further ahead
// than V (spills), instruction groups in fixed order 611 to 620 (606), wave priorities 632 (621), three
// waves a SIMD over a single V buffer 819 (601), loads spread over the step 584 to 591 (580). Eight waves on
// 256 rows 588 (604), which leaves fewer workgroups where rows are few.
template <typename E, int NK, bool FULL>
QMOE_DEV void many_rows(const AttentionArgs& a, int block, unsigned char* lds) {
  using L = Layout<NK>;
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Batch& batch = a.batch;
  // Heads next to each other (on XCDs of their own, whose L2 then holds few heads' keys), the last
  // tiles, which see the most keys, first; all first pieces before any second one, what there is not behind
  // all. An XCD's shader engines take workgroups in turn: with the pieces of a tile next to each other, most
  // of which there are not, all that there are went to one of the four (8000 new tokens 1978 us, now 620).
  const ManyList list(a);
  const int rest = a.heads.div(block), h = block - rest * a.Hkv;
  if (list.total == 0) return;
  const int piece = rest / list.total;
  if (piece >= a.pieces) return;
  const ManyTile mt = list.find(a, list.total - 1 - (rest - piece * list.total));
  if (mt.r0 < 0 || mt.r0 >= mt.rows) return;
  int t0 = 0, t1 = mt.tiles;
  bool cut = false;
  Pieces pieces = {};
  if (a.pieces > 1) {
    if (piece * 8 >= max(mt.tiles, 1)) return;  // no piece is shorter
    pieces = pieces_of(a, mt, h);
    const int count = piece_count(a, pieces, mt.tiles);
    if (piece >= count) return;
    cut = count > 1;
    const int each = (mt.tiles + count - 1) / count;
    t0 = min(piece * each, t1), t1 = min(t0 + each, t1);
  }
  const int G = a.group.d, b = mt.b, row0 = mt.row0, rows = mt.rows, r0 = mt.r0, before = mt.before, begin = mt.begin;
  const int end = min(before + (int)a.group.div(min(r0 + ROWS, rows) - 1) + 1, b < batch.B ? batch.length(b) : 0);

  const int r = r0 + 32 * wave + (lane & 31), token = a.group.div(r), of = r - token * G;
  const bool valid = r < rows;
  const long row = (long)(row0 + token) * a.Hq + h * G + of;  // of the output
  const int pos = before + token;
  const Seen seen = {a.window ? pos - a.window + 1 : 0, valid ? pos : -1};
  // the wave's first and last position
  const bool live = r0 + 32 * wave < rows;
  const int wave_first = before + (int)a.group.div(r0 + 32 * wave);
  const int wave_last = live ? before + (int)a.group.div(min(r0 + 32 * wave + 32, rows) - 1) : -1;

  s16x8_v q[2 * NK];  // the second operand of K Q^T: elements 16 ks + 8 half of row lane & 31
  const uint16_t* q_row = static_cast<const uint16_t*>(a.q) + (row0 + token) * a.q_token + (h * G + of) * a.q_head;
#pragma unroll
  for (int ks = 0; ks < 2 * NK; ++ks) q[ks] = q_piece(q_row, 16 * ks + 8 * half, a.D, valid, a.negate);
  Rows<E, NK, 1> acc;
  acc.clear();

  const unsigned char* kb = static_cast<const unsigned char*>(a.k) + 2 * h * a.kc.head;
  const unsigned char* vb = static_cast<const unsigned char*>(a.v) + 2 * h * a.vc.head;
  const int* table = batch.table + b * batch.table_ld;
  auto entry_of = [&](int tile) {
    const int key = begin + 64 * tile + lane;
    return key < end ? table[batch.page.div(key)] : -1;
  };
  // loads a tile, 1 KB at a time; returns which keys are there
  constexpr int GROUPS = 64 / L::RPI / 4;
  auto load = [&](int tile, int entry, unsigned char* to) {
    const int key = begin + 64 * tile + lane;
    if (entry >= batch.n_pages) entry = -1;
    const uint64_t present = __ballot(entry >= 0);
    const bool whole = present == ~0ull;
    const long ko = row_offset(a.kc, batch.page, entry, key), vo = row_offset(a.vc, batch.page, entry, key);
    to += 1024 * wave;
    load_rows<NK, FULL, GROUPS, 4 * L::RPI, true>(to, kb, ko, present, whole, a.same_pages, wave * L::RPI, (uint32_t)(2 * a.kc.slot), a.D);
    load_rows<NK, FULL, GROUPS, 4 * L::RPI, false>(to + L::TILE, vb, vo, present, whole, a.same_pages, wave * L::RPI,
                                                   (uint32_t)(2 * a.vc.slot), a.D);
    return present;
  };

  __shared__ int unusual;
  if (threadIdx.x == 0) unusual = 0;  // (before the first barrier of the loop, after which it may be set)
  __syncthreads();
  uint64_t present_next = 0;
  int entry = -1;
  if (t0 < t1) {
    present_next = load(t0, entry_of(t0), lds + (t0 & 1) * 2 * L::TILE);
    if (t0 + 1 < t1) entry = entry_of(t0 + 1);
  }
  const int k_row = lane & 31, k_base = k_row * L::STRIDE, k_swizzle = L::k_swizzle(k_row);
  const int last_pos = before + (int)a.group.div(min(r0 + ROWS, rows) - 1), first_pos = before + (int)a.group.div(r0);
  auto partial = [&](int tile, uint64_t present) {  // not seen whole by every row of the workgroup
    const int first = begin + 64 * tile;
    return present != ~0ull || first + 63 > first_pos || (a.window && first <= last_pos - a.window);
  };
  // One tile from LDS at `now`, while the next is loaded to `next`. As a function of two pointers that share
  // nothing, which spares a wait for the load before every transposing read; no wait and no barrier may stand
  // in it, which such pointers would let the reads pass.
  auto step = [&](int tile, const unsigned char* __restrict__ now, unsigned char* __restrict__ next) {
    const uint64_t present = present_next;
    if (tile + 1 < t1) {
      present_next = load(tile + 1, entry, next);
      if (tile + 2 < t1) entry = entry_of(tile + 2);
    }
    const int first = begin + 64 * tile;
    if (first > wave_last || (a.window && first + 63 <= wave_first - a.window)) return;
    // two halves of 32 keys: the matrix pipe takes the scores of the second while the vector pipe takes the
    // weights of the first, then the sums of the first while it takes the weights of the second
    f32x16_v s[2][1];
    auto score = [&](int j) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[j][0][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 2 * NK; ++ks) {
        u32x4_v f = *reinterpret_cast<const u32x4_v*>(now + k_base + 32 * j * L::STRIDE + 16 * ((2 * ks + half) ^ k_swizzle));
        if (!(FULL || L::always(ks) || 16 * ks + 8 * half < a.D)) f = (u32x4_v){0, 0, 0, 0};
        s[j][0] = Mma<E>::mma(__builtin_bit_cast(s16x8_v, f), q[ks], s[j][0]);
      }
    };
    const bool whole = present == ~0ull && first + 63 <= wave_first && (!a.window || first > wave_last - a.window);
    const unsigned char* v = now + L::TILE;
    s16x8_v p0[2], p1[2];
    score(0);
    if (!whole) acc.mask(s[0], seen, present, first);
    score(1);
    acc.settle(s[0], a.scale, p0, acc.weigh(s[0], a.scale, p0));
    if (!whole) acc.mask(s[1], seen, present >> 32, first + 32);
    acc.add(v, p0);
    acc.settle(s[1], a.scale, p1, acc.weigh(s[1], a.scale, p1));
    acc.add(v + 32 * L::STRIDE, p1);
  };
  for (int tile = t0; tile < t1; ++tile) {
    unsigned char *now = lds + (tile & 1) * 2 * L::TILE, *next = lds + (~tile & 1) * 2 * L::TILE;
    // the tile has landed, and every wave is past the one before it, whose half of LDS takes the next
    asm volatile("" ::: "memory");
    wait_vm_lgkm0<0>();
    if (partial(tile, present_next) && clean<E, GROUPS>(now + L::TILE + 1024 * wave, 4)) {
      unusual = 1;
      asm volatile("" ::: "memory");
      wait_vm_lgkm0<0>();
    }
    barrier_no_fence();
    step(tile, now, next);
  }
  __syncthreads();
  if (__builtin_expect(unusual, 0)) {
    for (int tile = t0; tile < t1; ++tile) {
      int e = entry_of(tile);
      if (e >= batch.n_pages) e = -1;
      const uint64_t present = __ballot(e >= 0);
      if (!partial(tile, present)) continue;
      const int key = begin + 64 * tile + lane;
      const long ko = row_offset(a.kc, batch.page, e, key), vo = row_offset(a.vc, batch.page, e, key);
#pragma unroll 1
      for (int j = 0; j < 2; ++j) {
        const int from = 32 * j + (lane & 31);
        acc.template add_unusual<FULL>(kb, __shfl(ko, from), vb, __shfl(vo, from), (uint32_t)(present >> (32 * j)), begin + 64 * tile + 32 * j, seen,
                        a.scale, [&](int ks) { return q[ks]; }, reinterpret_cast<float*>(lds) + 1024 * wave, a.D);
      }
    }
  }

  const float l = half_sum(acc.l);
  if (!valid) return;
  if (cut) {
    const long at = piece_at(a, pieces, piece) * ROWS + 32 * wave + (lane & 31);
    if (half == 0) many_tops(a)[at] = make_float2(acc.m, l);
    float* to = a.many_part + at * a.D;
#pragma unroll
    for (int dt = 0; dt < NK; ++dt)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = 32 * dt + 8 * c + 4 * half;
        if (d < a.D) *reinterpret_cast<f32x4_v*>(to + d) = (f32x4_v){acc.o[dt][4 * c], acc.o[dt][4 * c + 1], acc.o[dt][4 * c + 2], acc.o[dt][4 * c + 3]};
      }
    return;
  }
  if (l == 0.f) acc.clear();  // (also of a sum that a weight of 0 made NaN)
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* to = static_cast<uint16_t*>(a.out) + row * a.D;
#pragma unroll
  for (int dt = 0; dt < NK; ++dt)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int d = 32 * dt + 8 * c + 4 * half;
      if (d < a.D)
        *reinterpret_cast<uint2*>(to + d) = make_uint2(Mma<E>::pack(acc.o[dt][4 * c] * inv, acc.o[dt][4 * c + 1] * inv),
                                                       Mma<E>::pack(acc.o[dt][4 * c + 2] * inv, acc.o[dt][4 * c + 3] * inv));
    }
}

// ---------------------------------------------------------------- sequences of few rows

// A sequence of few rows: its keys [begin, end) and tiles of 128 of them, 0 for one that is not.
struct FewKeys {
  int n, before, begin, end, tiles;
};
QMOE_DEV FewKeys few_keys(const AttentionArgs& a, int b) {
  FewKeys s;
  s.n = a.batch.new_rows(b);
  s.before = tokens_before(a.batch, b, s.n);
  s.end = min(s.before + s.n, a.batch.length(b));
  s.begin = a.window ? max(s.before - a.window + 1, 0) & ~31 : 0;
  const bool is = s.n > 0 && s.n * (int)a.group.d <= a.few;
  s.tiles = is ? max(1, (max(s.end - s.begin, 0) + FEW_KEYS - 1) / FEW_KEYS) : 0;
  return s;
}

// The list of tiles: sequence, then head, then tile, with LEAD places before each head's tiles that stand for
// what a head costs beside them (its first loads and its sums through LDS, about as long as two tiles).
// Every workgroup takes `share` places.
constexpr int LEAD = 2;
struct FewList {
  FewKeys mine;  // of sequence `lane`
  int share;
  QMOE_DEV static int places(const FewKeys& k) { return k.tiles ? k.tiles + LEAD : 0; }
  QMOE_DEV FewList(const AttentionArgs& a) {
    const int lane = threadIdx.x & 63;
    mine = FewKeys{};
    if (lane < a.batch.B) mine = few_keys(a, lane);
    int sum = places(mine);
    for (int i = 64 + lane; i < a.batch.B; i += 64) sum += places(few_keys(a, i));
    const int total = lane_of(prefix_sum(sum), 63) * a.Hkv;
    share = max((total + a.few_blocks - 1) / a.few_blocks, 1);
  }
  // The sequence (B behind the end) that place f of the list belongs to, its keys and its first place.
  QMOE_DEV int locate(const AttentionArgs& a, int f, FewKeys& keys, int& start) const {
    const int lane = threadIdx.x & 63;
    start = 0;
    for (int i = 0; i < a.batch.B; i += 64) {
      FewKeys k = mine;
      if (i) k = i + lane < a.batch.B ? few_keys(a, i + lane) : FewKeys{};
      const int mine_all = places(k) * a.Hkv, upto = start + prefix_sum(mine_all);
      const uint64_t past = __ballot(upto > f);
      if (past) {
        const int at = __ffsll((unsigned long long)past) - 1;
        start = lane_of(upto - mine_all, at);
        keys = {lane_of(k.n, at), lane_of(k.before, at), lane_of(k.begin, at), lane_of(k.end, at), lane_of(k.tiles, at)};
        return i + at;
      }
      start = lane_of(upto, 63);
    }
    return a.batch.B;
  }
};
// Where a workgroup's part of a head's keys is kept: it has at most two that others share, one that
// it ends with and one that it goes on with.
QMOE_DEV long part_of(int block, bool begins) { return 2l * block + (begins ? 1 : 0); }

// A workgroup: its share of the list, tile by tile of 128 keys, each of its four waves 32 of them against all (up
// to 32) rows, K and V loaded to the wave's own quarter of LDS, so that waves meet only where a head ends. Each
// key is read once for all query heads of its group: bound by memory. 64 single tokens after up to 65536 (4 heads
// of 128, 1.29 GB) 248 us, 5.2 TB/s, 4 after 131072 (2 heads of 256, 1.07 GB) 190 us, 5.6; a kernel that
// only reads the same pages reached 5.6 to 6.0. 1 after 4096: 10 us, latency (a table entry, a key, sums), and 6
// to join its parts.
template <typename E, int NK, bool FULL>
QMOE_DEV void few_rows(const AttentionArgs& a, int block, unsigned char* lds) {
  using L = Layout<NK>;
  __shared__ float m_of[4][32], l_of[4][32];
  __shared__ s16x8_v q_lds[NK > 4 ? 2 * NK * 64 : 1];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Batch& batch = a.batch;
  const int G = a.group.d;

  if (!a.many_tiles) {  // rows behind the last sequence
    const long from = (long)batch.start(batch.B) * a.Hq * a.D / 8, to = (long)batch.T * a.Hq * a.D / 8;
    for (long i = from + block * 256l + threadIdx.x; i < to; i += a.few_blocks * 256l)
      static_cast<u32x4_v*>(a.out)[i] = (u32x4_v){0, 0, 0, 0};
  }

  const FewList list(a);
  const int stop = list.share * (block + 1);
  int f = list.share * block, start;
  FewKeys keys;
  int b = list.locate(a, f, keys, start);
  while (f < stop && b < batch.B) {
    const int each = FewList::places(keys), h = (f - start) / each, tiles_start = start + h * each + LEAD;
    const int x0 = max(f - tiles_start, 0), x1 = min(keys.tiles, stop - tiles_start);
    f = tiles_start + max(x1, 0);
    if (x1 <= 0) break;  // its places before the tiles only
    const int row0 = batch.first_row(b), rows = keys.n * G;

    const int r = lane & 31, token = a.group.div(r), of = r - token * G;
    const bool valid = r < rows;
    const int pos = keys.before + token;
    const Seen seen = {a.window ? pos - a.window + 1 : 0, valid ? pos : -1};
    // q in registers, or, where the sums of wide heads need these, in LDS
    s16x8_v q[NK > 4 ? 1 : 2 * NK];
    const uint16_t* q_row = static_cast<const uint16_t*>(a.q) + (row0 + token) * a.q_token + (h * G + of) * a.q_head;
    if constexpr (NK > 4) {
#pragma unroll
      for (int ks = wave; ks < 2 * NK; ks += 4) q_lds[ks * 64 + lane] = q_piece(q_row, 16 * ks + 8 * half, a.D, valid, a.negate);
      __syncthreads();
    } else {
#pragma unroll
      for (int ks = 0; ks < 2 * NK; ++ks) q[ks] = q_piece(q_row, 16 * ks + 8 * half, a.D, valid, a.negate);
    }
    Rows<E, NK, 1> acc;
    acc.clear();

    const unsigned char* kb = static_cast<const unsigned char*>(a.k) + 2 * h * a.kc.head;
    const unsigned char* vb = static_cast<const unsigned char*>(a.v) + 2 * h * a.vc.head;
    const int* table = batch.table + b * batch.table_ld;
    auto first_of = [&](int x) { return keys.begin + FEW_KEYS * x + 32 * wave; };
    auto entry_of = [&](int x) {
      const int key = first_of(x) + (lane & 31);
      return x < x1 && key < keys.end ? table[batch.page.div(key)] : -1;
    };
    unsigned char* mine = lds + wave * 64 * L::STRIDE;  // two times 32 rows of V
    auto within = [&](int ks) { return FULL || L::always(ks) || 16 * ks + 8 * half < a.D; };
    // K's rows go straight to registers (lane & 31 is the row of the first operand), V's to LDS
    s16x8_v k[2 * NK];
    auto load_k = [&](int x, int entry) {
      // (a key without a page: the cache's first, left out by its score)
      const unsigned char* row = kb + row_offset(a.kc, batch.page, entry, first_of(x) + (lane & 31));
#pragma unroll
      for (int ks = 0; ks < 2 * NK; ++ks) k[ks] = *reinterpret_cast<const s16x8_v*>(row + (within(ks) ? 32 * ks + 16 * half : 0));
    };
    // The elements behind a head's: others of its row, made 0 where they are used, as at the load that would
    // wait for them.
    auto key_part = [&](int ks) {
      u32x4_v w = __builtin_bit_cast(u32x4_v, k[ks]);
      if (!within(ks)) w = (u32x4_v){0, 0, 0, 0};
      return __builtin_bit_cast(s16x8_v, w);
    };
    auto load_v = [&](int x, int entry, uint64_t present, unsigned char* to) {
      const long vo = row_offset(a.vc, batch.page, entry, first_of(x) + (lane & 31));
      load_rows<NK, FULL, 32 / L::RPI, L::RPI, false>(to, vb, vo, present, present == ~0ull, a.same_pages, 0, (uint32_t)(2 * a.vc.slot), a.D);
    };
    uint64_t present = 0;
    int entry = entry_of(x0), entry_next = entry_of(x0 + 1);
    auto known = [&](int e) { return e < batch.n_pages ? e : -1; };
    entry = known(entry);
    present = __ballot(entry >= 0);
    const bool any = keys.end > keys.begin;  // (there is a page, then)
    if (any) {
      load_v(x0, entry, present, mine);
      load_k(x0, entry);
    }
    bool unusual = false;
    auto whole = [&](int x, uint64_t there) {  // seen by every row
      const int first = first_of(x);
      return there == ~0ull && first + 31 <= keys.before && (!a.window || first > keys.before + keys.n - 1 - a.window);
    };
    // One tile's V in LDS at `v`, while the next is loaded to `next` (no wait in it, as in the other form).
    auto step = [&](int x, const unsigned char* __restrict__ v, unsigned char* __restrict__ next) {
      const uint64_t here = present;
      entry = known(entry_next);
      present = __ballot(entry >= 0);
      if (x + 1 < x1) load_v(x + 1, entry, present, next);
      entry_next = entry_of(x + 2);
      const int first = first_of(x);
      f32x16_v s[1];
#pragma unroll
      for (int i = 0; i < 16; ++i) s[0][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 2 * NK; ++ks) {
        if constexpr (NK > 4) s[0] = Mma<E>::mma(key_part(ks), q_lds[ks * 64 + lane], s[0]);
        else s[0] = Mma<E>::mma(key_part(ks), q[ks], s[0]);
      }
      // The next keys take these registers (behind the last tile: the first row of the cache; a branch around
      // the loads would cost a wait for them where it ends).
      asm volatile("" ::: "memory");
      load_k(x + 1, entry);
      if (!whole(x, here)) acc.mask(s, seen, here, first);
      s16x8_v p[2];
      acc.settle(s, a.scale, p, acc.weigh(s, a.scale, p));
      acc.add(v, p);
    };
    for (int x = x0; any && x < x1; ++x) {
      unsigned char *v = mine + ((x - x0) & 1) * 32 * L::STRIDE, *next = mine + ((x - x0 + 1) & 1) * 32 * L::STRIDE;
      asm volatile("" ::: "memory");
      wait_vm_lgkm0<0>();
      asm volatile("" ::: "memory");
      if (!whole(x, present) && clean<E, 32 / L::RPI>(v, 1)) unusual = true;
      step(x, v, next);
    }
    if (__builtin_expect(unusual, 0)) {
      for (int x = x0; x < x1; ++x) {
        const int e = known(entry_of(x));
        const uint64_t there = __ballot(e >= 0);
        if (whole(x, there)) continue;
        const int key = first_of(x) + (lane & 31);
        acc.template add_unusual<FULL>(kb, row_offset(a.kc, batch.page, e, key), vb, row_offset(a.vc, batch.page, e, key), (uint32_t)there,
                        first_of(x), seen, a.scale, [&](int ks) { return NK > 4 ? q_lds[ks * 64 + lane] : q[NK > 4 ? 0 : ks]; },
                        reinterpret_cast<float*>(mine), a.D);
      }
    }

    // the four waves' sums: each brought to the common maximum, then added through LDS
    const float l = half_sum(acc.l);
    if (half == 0) m_of[wave][r] = acc.m, l_of[wave][r] = l;
    __syncthreads();  // (and V's rows in LDS are done with)
    float top = m_of[0][r];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, m_of[w][r]);
    const float scale = acc.m == top ? 1.f : __builtin_amdgcn_exp2f(acc.m - top);
    f32x4_v* sums = reinterpret_cast<f32x4_v*>(lds) + (wave * 32 + r) * (L::DC / 4);
#pragma unroll
    for (int dt = 0; dt < NK; ++dt)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        sums[(8 * dt + 2 * c + half) ^ (r & 7)] = (f32x4_v){acc.o[dt][4 * c] * scale, acc.o[dt][4 * c + 1] * scale,
                                                            acc.o[dt][4 * c + 2] * scale, acc.o[dt][4 * c + 3] * scale};
    __syncthreads();
    const bool alone = x0 == 0 && x1 == keys.tiles;
    const long part = part_of(block, x0 == 0);
    const int quads = a.D / 4;
    for (int i = threadIdx.x; i < rows * quads; i += 256) {
      const int at = i / quads, d = i - at * quads;
      float best = m_of[0][at], total = 0.f;
#pragma unroll
      for (int w = 1; w < 4; ++w) best = fmaxf(best, m_of[w][at]);
      f32x4_v sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        sum += reinterpret_cast<const f32x4_v*>(lds)[(w * 32 + at) * (L::DC / 4) + (d ^ (at & 7))];
        total += l_of[w][at] * (m_of[w][at] == best ? 1.f : __builtin_amdgcn_exp2f(m_of[w][at] - best));
      }
      if (alone) {
        if (total == 0.f) sum = (f32x4_v){0.f, 0.f, 0.f, 0.f};
        const float inv = total == 0.f ? 0.f : 1.f / total;
        const int tok = a.group.div(at);
        const long row = (long)(row0 + tok) * a.Hq + h * G + at - tok * G;
        reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + row * a.D)[d] =
            make_uint2(Mma<E>::pack(sum[0] * inv, sum[1] * inv), Mma<E>::pack(sum[2] * inv, sum[3] * inv));
      } else {
        reinterpret_cast<f32x4_v*>(a.few_part + (part * a.few_rows + at) * a.D)[d] = sum;
        if (d == 0) few_tops(a)[part * a.few_rows + at] = make_float2(best, total);
      }
    }
    __syncthreads();
    if (f >= start + each * a.Hkv && f < stop) b = list.locate(a, f, keys, start);
  }
}

// Each form by itself, and both in one launch: few rows' equal shares in the last blocks, where they fill what
// the other form's tiles leave (8 sequences of up to 500 after up to 30000 365 us, 393 in the first), or in the
// first, where most sequences must be of few rows (16 of up to 5 tokens 24.5 us, 29.9 in the last).
// Heads of 64 in few rows alone: three workgroups on a CU, with 168 registers a wave.
enum { MANY = 1, FEW_ROWS = 2 };
template <typename E, int NK, bool FULL, int FORMS>
__global__ __launch_bounds__(256, (NK == 2 && FULL && FORMS == FEW_ROWS ? 3 : NK <= 4 ? 2 : 1)) void attention_kernel(AttentionArgs a) {
  __shared__ __align__(16) unsigned char lds[Layout<NK>::LDS];
  if constexpr (FORMS == MANY) many_rows<E, NK, FULL>(a, blockIdx.x, lds);
  else if constexpr (FORMS == FEW_ROWS) few_rows<E, NK, FULL>(a, blockIdx.x, lds);
  else if (blockIdx.x - a.few_from < (unsigned)a.few_blocks) few_rows<E, NK, FULL>(a, blockIdx.x - a.few_from, lds);
  else many_rows<E, NK, FULL>(a, blockIdx.x - (a.few_from ? 0 : a.few_blocks), lds);
}

// ---------------------------------------------------------------- joining

// Rows' parts: sums of D and (maximum, sum), `count` of them for a row, part c of row r at at(r, c); rows
// `from` and so on below `rows`. Up to 64 parts: a wave to a row; more: a workgroup to a row; `slots`
// workgroups share the rows. The parts' scales first, then as many parts at once as threads make rows of D, eight of
// them in flight each.
static_assert(FEW_BLOCKS_MAX <= 3 * 256);
template <typename E, typename At, typename Out>
QMOE_DEV void join_rows(const float* sums, const float2* tops, At at, int count, int slot, int slots, int rows, Out out, int D) {
  __shared__ float scale[FEW_BLOCKS_MAX], sum_of[4];
  __shared__ __align__(16) f32x4_v part[256];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const bool alone = count <= 64;  // a wave by itself
  const int tid = alone ? lane : threadIdx.x, threads = alone ? 64 : 256;
  const int quads = D / 4, streams = threads / quads, stream = tid / quads, quad = tid - stream * quads;
  float* scales = alone ? scale + 64 * wave : scale;
  f32x4_v* parts = alone ? part + 64 * wave : part;
  auto meet = [&] {
    if (alone) wave_fence();
    else __syncthreads();
  };
  for (int r = alone ? slot * 4 + wave : slot; r < rows; r += alone ? 4 * slots : slots) {
    float2 t[3];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      t[i] = make_float2(-INFINITY, 0.f);
      if ((i == 0 || !alone) && tid + 256 * i < count) t[i] = tops[at(r, tid + 256 * i)];
      m = fmaxf(m, t[i].x);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (!alone) {
      if (lane == 0) sum_of[wave] = m;
      meet();
      m = fmaxf(fmaxf(sum_of[0], sum_of[1]), fmaxf(sum_of[2], sum_of[3]));
      meet();
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if ((i == 0 || !alone) && tid + 256 * i < count) {
        const float f = t[i].x == m ? 1.f : __builtin_amdgcn_exp2f(t[i].x - m);
        scales[tid + 256 * i] = f;
        l += t[i].y * f;
      }
    l = wave_sum_f32(l);
    if (!alone && lane == 0) sum_of[wave] = l;
    meet();
    if (!alone) l = (sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3]);
    f32x4_v o = {0.f, 0.f, 0.f, 0.f};
    if (stream < streams)
      for (int c = stream; c < count; c += 8 * streams) {
        f32x4_v x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = reinterpret_cast<const f32x4_v*>(sums + at(r, min(c + i * streams, count - 1)) * D)[quad];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i * streams < count) o += x[i] * scales[c + i * streams];
      }
    parts[tid] = o;
    meet();
    if (tid < quads) {
      for (int c = 1; c < streams; ++c) o += parts[c * quads + tid];
      if (l == 0.f) o = (f32x4_v){0.f, 0.f, 0.f, 0.f};
      const float inv = l == 0.f ? 0.f : 1.f / l;
      reinterpret_cast<uint2*>(out(r))[tid] = make_uint2(Mma<E>::pack(o[0] * inv, o[1] * inv), Mma<E>::pack(o[2] * inv, o[3] * inv));
    }
    meet();
  }
}

// Blocks [0, few_blocks) x join_few: the head inside whose tiles the first boundary is the one between the
// shares of block - 1 and block. Behind them, where the many-rows form cuts keys into pieces, join_many
// for each tile and head.
template <typename E>
__global__ __launch_bounds__(256) void join_kernel(AttentionArgs a) {
  const Batch& batch = a.batch;
  const int few = a.few_blocks * a.join_few, G = a.group.d;
  const bool is_few = (int)blockIdx.x < few;
  const int slots = is_few ? a.join_few : a.join_many, at = is_few ? blockIdx.x : blockIdx.x - few, block = at / slots, slot = at - block * slots;
  const float *sums, *tops;
  int count, rows, row0, h, first;  // rows of the tile; its first token's row and its own first row
  Pieces pieces = {};
  if (is_few) {
    if (block == 0) return;
    const FewList list(a);
    const int f = list.share * block;
    FewKeys keys;
    int start;
    const int b = list.locate(a, f, keys, start);
    if (b >= batch.B) return;
    const int each = FewList::places(keys);
    h = (f - start) / each;
    start += h * each + LEAD;
    if (start >= f || start < f - list.share) return;
    count = (start + keys.tiles - 1) / list.share - block + 2;
    rows = keys.n * G, row0 = batch.first_row(b), first = 0;
  } else {
    const int number = a.heads.div(block);
    h = block - number * a.Hkv;
    const ManyList list(a);
    if (number >= list.total) return;
    const ManyTile t = list.find(a, number);
    if (t.r0 < 0 || t.r0 >= t.rows || t.tiles <= whole_tiles(a.D)) return;
    pieces = pieces_of(a, t, h);
    count = piece_count(a, pieces, t.tiles);
    if (count <= 1) return;
    rows = min(ROWS, t.rows - t.r0), row0 = t.row0, first = t.r0;
  }
  sums = is_few ? a.few_part : a.many_part;
  tops = reinterpret_cast<const float*>(is_few ? few_tops(a) : many_tops(a));
  join_rows<E>(sums, reinterpret_cast<const float2*>(tops),
               [&](int r, int c) { return is_few ? part_of(block - 1 + c, c == 0) * a.few_rows + r : piece_at(a, pieces, c) * ROWS + r; },
               count, slot, slots, rows,
               [&](int r) {
                 const int token = a.group.div(first + r);
                 const long row = (long)(row0 + token) * a.Hq + h * G + first + r - token * G;
                 return static_cast<uint16_t*>(a.out) + row * a.D;
               },
               a.D);
}

// ---------------------------------------------------------------- host

// How a call is cut, from what the host knows of it: sequences are taken to be as long as the table is wide. A wide table thus
// brings pieces, their workspace and a joining launch that the device then has no use for. us with a table as wide as
// the prompt, and of 131072 tokens: 32 over 8 heads of 128, prompts of 512 20.8, 28.1, 1024 34.0, 40.5, 2048 64.4,
// 63.3, 4096 165, 162; 16 over 2 of 256, 1024 58.6, 63.1, 2048 106.6, 106.8; 256 after 3000 46.8, 46.8.
struct Plan {
  int few, few_blocks, few_rows, many_tiles, pieces, slots;
  size_t few_floats, many_floats;
};
constexpr int PIECES_MAX = 64;
Plan plan_for(int T, int B, int Hq, int Hkv, int D, int page, int width, int window, bool one_each) {
  const int G = Hq / Hkv;
  Plan p = {};
  const bool many = one_each ? G > FEW : (long)T * G > FEW;  // may there be sequences of many rows
  const bool few = !many || (!one_each && B > 1);            // and of few
  p.few = few ? FEW : 0;
  p.few_rows = one_each ? G : FEW;
  p.pieces = 1;
  p.slots = D > 128 ? 256 : 512;  // workgroups that run at once
  const long most = (long)width * page;  // keys
  if (few) {
    const long tiles = (long)B * Hkv * (std::max<long>(1, (most + FEW_KEYS - 1) / FEW_KEYS));
    // Heads of 64 by themselves leave registers and LDS for three workgroups on a CU (4 tokens after 65536 128 us
    // with two, 108 with three, 64 after up to 16384 83, 78); beside the other form's tiles they gain nothing.
    p.few_blocks = (int)std::max(1l, std::min<long>(D == 64 && !many ? FEW_BLOCKS_MAX : p.slots, tiles));
    p.few_floats = 2l * p.few_blocks * p.few_rows * (D + 2);
  }
  if (many) {
    // a tile for 128 rows, and one more that is not full for each such sequence and for the rows behind the last
    const long rows = (long)T * G;
    p.many_tiles = (int)(rows / ROWS + std::min<long>(B, few ? rows / (FEW + 1) : B) + 1);
    const long items = (rows + ROWS - 1) / ROWS * Hkv;
    const long units = (most + 63) / 64, seen = window ? std::min(units, (window + ROWS / G + 127l) / 64) : units;
    // What pieces may save, in steps of a workgroup. One sequence: up to a tile on each workgroup, what all of them
    // are short of the longest; more tiles, longest first, what the last round of the shortest is short of workgroups.
    // us in pieces and whole: prompts of 1024 54, 34, of 2048 74, 64, of 4096 187, 164; 256 tokens after 2048 39, 61,
    // 1024 after 8192 197, 226. (A window never adds pieces: the workspace is asked for without it.)
    auto gain = [&](long longest, long shortest) {
      if (B > 1) return longest;
      return items <= p.slots ? longest - items * (longest + shortest) / (2 * p.slots)
                              : shortest * ((p.slots - items % p.slots) % p.slots) / p.slots;
    };
    const long gains = std::min(gain(units, std::max(units - T / 64, 0l)), window ? gain(seen, seen) : units);
    if (items < 4 * p.slots && gains > whole_tiles(D) && ((long)p.many_tiles * Hkv + 2 * p.slots) * (units + 8) < 1l << 31)
      p.pieces = (int)std::max<long>(1, std::min({seen / 8, (long)PIECES_MAX, std::max(8l, 16l * p.slots / items)}));
    if (p.pieces > 1) p.many_floats = 2l * (2 * p.slots + 1) * ROWS * (D + 2);
  }
  return p;
}

template <typename E, int NK, bool FULL>
int launch(const AttentionArgs& a, hipStream_t st) {
  const long tiles = (long)a.many_tiles * a.Hkv, blocks = tiles * a.pieces + a.few_blocks;
  const dim3 grid((unsigned)blocks), threads(256);
  if (!a.few_blocks) hipLaunchKernelGGL((attention_kernel<E, NK, FULL, MANY>), grid, threads, 0, st, a);
  else if (!tiles) hipLaunchKernelGGL((attention_kernel<E, NK, FULL, FEW_ROWS>), grid, threads, 0, st, a);
  else hipLaunchKernelGGL((attention_kernel<E, NK, FULL, MANY | FEW_ROWS>), grid, threads, 0, st, a);
  const int rc = (int)hipGetLastError();
  const long joins = (long)a.few_blocks * a.join_few + (a.pieces > 1 ? tiles * a.join_many : 0);
  if (rc || joins == 0) return rc;
  hipLaunchKernelGGL((join_kernel<E>), dim3((unsigned)joins), threads, 0, st, a);
  return (int)hipGetLastError();
}

template <typename E, int NK>
int launch_heads(const AttentionArgs& a, hipStream_t st) {
  return a.D == 32 * NK ? launch<E, NK, true>(a, st) : launch<E, NK, false>(a, st);
}

template <typename E>
int dispatch(const AttentionArgs& a, hipStream_t st) {
  switch (blocks_of(a.D)) {
    case 2: return launch_heads<E, 2>(a, st);
    case 3: return launch_heads<E, 3>(a, st);
    case 4: return launch_heads<E, 4>(a, st);
    case 6: return launch_heads<E, 6>(a, st);
  }
  return launch_heads<E, 8>(a, st);
}

bool bad_shape(int T, int B, int Hq, int Hkv, int D) {
  return T < 0 || B < 0 || Hq < 1 || Hkv < 1 || Hq > 4096 || Hq % Hkv || Hq / Hkv > GROUP_MAX || D < 8 || D > D_MAX || D % 8 ||
         (long)T * Hq > 0x7fffffffl;
}

}  // namespace

extern "C" {

size_t qmoe_paged_attention_workspace(int T, int B, int Hq, int Hkv, int D, int page, int table_width, int one_each) {
  if (bad_shape(T, B, Hq, Hkv, D) || page < 1 || table_width < 0 || (long)table_width * page > TOKENS_MAX) return 0;
  const Plan p = plan_for(T, B, Hq, Hkv, D, page, table_width, 0, one_each);
  return 4 * (p.few_floats + p.many_floats);
}

int qmoe_paged_attention(const void* q, long q_token, long q_head, const void* k_cache, long k_page, long k_slot,
                         long k_head, const void* v_cache, long v_page, long v_slot, long v_head, int type,
                         const void* table, long table_ld, int table_width, const void* lengths, const void* starts,
                         void* out, int T, int B, int Hq, int Hkv, int D, int page, long n_pages, float scale,
                         int window, void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_shape(T, B, Hq, Hkv, D) || (type != QMOE_BF16 && type != QMOE_F16)) return QMOE_EINVAL;
  constexpr float LOG2E = 1.44269504088896341f;
  if (page < 1 || page > 1 << 30 || n_pages < 0 || table_width < 0 || table_ld < 0 || (!starts && T != B) ||
      window < 0 || window > 1 << 30 || !std::isfinite(scale * LOG2E) || (long)table_width * page > TOKENS_MAX)
    return QMOE_EINVAL;
  if ((k_page | k_slot | k_head | v_page | v_slot | v_head) & 7) return QMOE_EINVAL;
  if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) return QMOE_EINVAL;
  // bytes within a page, from page to page, and the list of the few-rows form (rounded up to equal shares) are
  // counted in 32 bits
  for (const long step : {k_page, v_page, k_slot * page, v_slot * page, k_head, v_head})
    if (step < 0 || step >= 1l << 30) return QMOE_EINVAL;
  if ((long)B * Hkv > (0x7fffffffl - FEW_BLOCKS_MAX) / ((long)table_width * page / FEW_KEYS + 1 + LEAD)) return QMOE_EINVAL;
  if (T == 0) return QMOE_OK;
  if (!q || !out || missing(k_cache, v_cache, n_pages, table, table_width, lengths, B)) return QMOE_EINVAL;
  const Plan p = plan_for(T, B, Hq, Hkv, D, page, table_width, window, !starts);
  // a grid holds fewer than 2^32 threads
  if ((long)p.many_tiles * Hkv * p.pieces + p.few_blocks >= (1l << 32) / 256) return QMOE_EINVAL;
  if (p.few_floats + p.many_floats &&
      (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < 4 * (p.few_floats + p.many_floats)))
    return QMOE_EWORKSPACE;
  AttentionArgs a = {};
  a.q = q, a.k = k_cache, a.v = v_cache, a.out = out, a.q_token = q_token, a.q_head = q_head;
  a.kc = {k_page, k_slot, k_head}, a.vc = {v_page, v_slot, v_head};
  a.batch.table = static_cast<const int*>(table), a.batch.lengths = static_cast<const int*>(lengths);
  a.batch.starts = static_cast<const int*>(starts);
  a.batch.table_ld = table_ld, a.batch.n_pages = n_pages, a.batch.T = T, a.batch.B = B, a.batch.width = table_width;
  a.batch.page = FastDiv(page);
  a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.window = window;
  a.group = FastDiv(Hq / Hkv), a.heads = FastDiv(Hkv);
  a.scale = std::max(std::fabs(scale) * LOG2E, FLT_MIN), a.negate = scale < 0;
  a.same_pages = page % 16 == 0;
  a.few = p.few, a.few_blocks = p.few_blocks, a.few_rows = p.few_rows, a.many_tiles = p.many_tiles;
  a.pieces = p.pieces, a.slots = p.slots;
  a.few_from = (long)T * (Hq / Hkv) <= (long)B * FEW ? 0 : p.many_tiles * Hkv * p.pieces;
  // few heads: parts of a row beyond 64, a workgroup to each row
  a.join_few = p.few_blocks > 48l * B * Hkv ? 8 : 2;
  // Few tiles: most are in pieces, and more workgroups join them sooner; many: most are not, and the workgroups
  // are in the way. 4, 8, 16, 32 for each, us: 16 tiles 83, 69, 61, 59, 264 189, 177, 171, 176, 707 (none in
  // pieces) 84, 88, 99, 118.
  const long items = ((long)T * (Hq / Hkv) + ROWS - 1) / ROWS * Hkv;
  a.join_many = items <= 32 ? 32 : items <= 384 ? 16 : items <= 640 ? 8 : 4;
  a.few_part = static_cast<float*>(workspace);
  a.many_part = a.few_part + p.few_floats;
  return type == QMOE_BF16 ? dispatch<ElemBF16>(a, (hipStream_t)stream) : dispatch<ElemF16>(a, (hipStream_t)stream);
}

}  // extern "C"
