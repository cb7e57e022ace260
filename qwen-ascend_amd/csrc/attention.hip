// Attention of new tokens over the pages of their sequences.
//
// Row (t, h) at position p of its sequence sees the keys j with p - window < j <= p that lie on a
// page of the cache:  o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale * q.k_j,
// m = max_j s_j. Scores, sums and the output's sums in fp32, one rounding at the end. A row that
// sees no key, or whose scores are all -inf, gives 0.
#include "paged.h"

#include <cmath>

namespace {

struct AttentionArgs {
  const void *q, *k, *v;
  void* out;
  long q_token, q_head;
  CacheSteps kc, vc;
  Batch batch;
  int Hq, Hkv, group, D, window;
  float scale;
};

// One wave per row: its lanes hold the elements of a head, one key after the other.
template <typename E>
__global__ __launch_bounds__(256) void attention_rows_kernel(AttentionArgs a) {
  using raw = typename E::raw;
  const int lane = threadIdx.x & 63;
  const long row = blockIdx.x * 4l + (threadIdx.x >> 6);
  if (row >= (long)a.batch.T * a.Hq) return;
  const int t = (int)(row / a.Hq), h = (int)(row - (long)t * a.Hq), kv = h / a.group;
  float q[4] = {}, o[4] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < a.D) q[i] = E::load(static_cast<const raw*>(a.q)[t * a.q_token + h * a.q_head + lane + 64 * i]);
  const int b = a.batch.sequence(t);
  if (b < a.batch.B) {
    const long p = (long)a.batch.lengths[b] - a.batch.new_rows(b) + t - a.batch.first_row(b);
    const int end = (int)min(p + 1, (long)a.batch.length(b)), begin = a.window ? (int)max(p - a.window + 1, 0l) : 0;
    for (int j = begin; j < end; ++j) {
      const long page = a.batch.page_of(b, j);
      if (page < 0) continue;
      const int slot = j - (int)a.batch.page.div(j) * (int)a.batch.page.d;
      const raw* k = static_cast<const raw*>(a.k) + page * a.kc.page + slot * a.kc.slot + kv * a.kc.head;
      const raw* v = static_cast<const raw*>(a.v) + page * a.vc.page + slot * a.vc.slot + kv * a.vc.head;
      float s = 0.f, x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = 0.f;
        if (lane + 64 * i < a.D) s += q[i] * E::load(k[lane + 64 * i]), x[i] = E::load(v[lane + 64 * i]);
      }
      s = wave_sum_f32(s) * a.scale;
      if (s == -INFINITY) continue;
      if (s > m) {
        const float c = expf(m - s);
        l *= c, m = s;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= c;
      }
      const float e = expf(s - m);
      l += e;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] += e * x[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < a.D) static_cast<raw*>(a.out)[row * a.D + lane + 64 * i] = E::store(l == 0.f ? 0.f : o[i] / l);
}

template <typename E>
int launch(const AttentionArgs& a, hipStream_t st) {
  const long rows = (long)a.batch.T * a.Hq;
  hipLaunchKernelGGL((attention_rows_kernel<E>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

constexpr int D_MAX = 256, GROUP_MAX = 64;

bool bad_shape(int T, int B, int Hq, int Hkv, int D) {
  return T < 0 || B < 0 || Hq < 1 || Hkv < 1 || Hq > 4096 || Hq % Hkv || Hq / Hkv > GROUP_MAX || D < 8 || D > D_MAX || D % 8 ||
         (long)T * Hq > 0x7fffffffl;
}

}  // namespace

extern "C" {

size_t qmoe_paged_attention_workspace(int T, int B, int Hq, int Hkv, int D, int page, int table_width, int one_each) {
  return 0;
}

int qmoe_paged_attention(const void* q, long q_token, long q_head, const void* k_cache, long k_page, long k_slot,
                         long k_head, const void* v_cache, long v_page, long v_slot, long v_head, int type,
                         const void* table, long table_ld, int table_width, const void* lengths, const void* starts,
                         void* out, int T, int B, int Hq, int Hkv, int D, int page, long n_pages, float scale,
                         int window, void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_shape(T, B, Hq, Hkv, D) || (type != QMOE_BF16 && type != QMOE_F16)) return QMOE_EINVAL;
  if (page < 1 || page > 1 << 30 || n_pages < 0 || table_width < 0 || table_ld < 0 || (!starts && T != B) ||
      window < 0 || !std::isfinite(scale))
    return QMOE_EINVAL;
  if ((k_page | k_slot | k_head | v_page | v_slot | v_head) & 7) return QMOE_EINVAL;
  if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) return QMOE_EINVAL;
  if (T == 0) return QMOE_OK;
  if (!q || !out || missing(k_cache, v_cache, n_pages, table, table_width, lengths, B)) return QMOE_EINVAL;
  AttentionArgs a = {};
  a.q = q, a.k = k_cache, a.v = v_cache, a.out = out, a.q_token = q_token, a.q_head = q_head;
  a.kc = {k_page, k_slot, k_head}, a.vc = {v_page, v_slot, v_head};
  a.batch.table = static_cast<const int*>(table), a.batch.lengths = static_cast<const int*>(lengths);
  a.batch.starts = static_cast<const int*>(starts);
  a.batch.table_ld = table_ld, a.batch.n_pages = n_pages, a.batch.T = T, a.batch.B = B, a.batch.width = table_width;
  a.batch.page = FastDiv(page);
  a.Hq = Hq, a.Hkv = Hkv, a.group = Hq / Hkv, a.D = D, a.window = window, a.scale = scale;
  return type == QMOE_BF16 ? launch<ElemBF16>(a, (hipStream_t)stream) : launch<ElemF16>(a, (hipStream_t)stream);
}

}  // extern "C"
