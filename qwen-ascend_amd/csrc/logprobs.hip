// Log probabilities of given tokens, entropy and top alternatives of rows of logits.
//
//   Z = sum_v e^l_v;  logprob(v) = l_v - ln Z;  entropy = -sum_v p_v ln p_v
//
// over the allowed v, from m = max l, S = sum e^(l - m), D = sum e^(l - m) (l - m) (base 2
// inside): logprob(v) = (l_v - m) - ln S, entropy = ln S - D / S. Sums in fp32.
#include "elem_types.h"

#include <algorithm>

namespace {

constexpr int TOP_MAX = 32;
constexpr int THREADS = 256, WAVES = THREADS / 64;
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

QMOE_DEV Part join(Part a, Part b) {
  const float m = fmaxf(a.m, b.m), z = base_of(m);
  const float da = (a.m - z) * LOG2E, db = (b.m - z) * LOG2E;
  const float ca = __builtin_amdgcn_exp2f(da), cb = __builtin_amdgcn_exp2f(db);
  Part r;
  r.m = m;
  r.s = ca * a.s + cb * b.s;
  r.d = ca * (a.d + fmaxf(da, FAR) * a.s) + cb * (b.d + fmaxf(db, FAR) * b.s);
  return r;
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

template <typename E>
__global__ __launch_bounds__(THREADS) void logprob_rows_kernel(LogprobArgs a) {
  __shared__ Part part[WAVES];
  __shared__ uint64_t best[WAVES];
  for (int t = blockIdx.x; t < a.T; t += gridDim.x) {
    const auto* x = static_cast<const typename E::raw*>(a.logits) + (long)t * a.ld;
    const uint8_t* ok = a.allowed ? a.allowed + (long)t * a.lda : nullptr;
    auto logit = [&](int v) { return (ok && !ok[v]) ? -INFINITY : E::load(x[v]); };
    Part p = {-INFINITY, 0.f, 0.f};
    for (int v = threadIdx.x; v < a.V; v += THREADS) p = join(p, {logit(v), 1.f, 0.f});
#pragma unroll
    for (int o = 32; o; o >>= 1) p = join(p, {__shfl_xor(p.m, o), __shfl_xor(p.s, o), __shfl_xor(p.d, o)});
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = p;
    __syncthreads();
    p = part[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) p = join(p, part[w]);
    const bool undefined = !(p.s >= 0.f);  // a NaN or +inf at an allowed place
    const float log_s = logf(p.s);
    if (threadIdx.x == 0) a.entropy[t] = p.s == 0.f ? 0.f : log_s - LN2 * p.d / p.s;
    for (int j = threadIdx.x; j < a.m; j += THREADS) {
      const int64_t tok = a.tokens[(long)t * a.m + j];
      float r = 0.f;
      if (tok >= a.V || undefined) r = NAN;
      else if (tok >= 0) {
        const float l = logit((int)tok);
        r = l == -INFINITY ? l : (l - p.m) - log_s;
      }
      a.logprobs[(long)t * a.m + j] = tok < 0 ? 0.f : r;
    }
    uint64_t last = ~0ull;
    for (int j = 0; j < a.top; ++j) {
      uint64_t k = 0;
      for (int v = threadIdx.x; v < a.V; v += THREADS) {
        const float l = logit(v);
        const uint64_t q = l > -INFINITY ? key_of(l, v) : 0;
        if (q < last && q > k) k = q;
      }
#pragma unroll
      for (int o = 32; o; o >>= 1) k = max(k, (uint64_t)__shfl_xor((unsigned long long)k, o));
      __syncthreads();
      if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = k;
      __syncthreads();
      k = best[0];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) k = max(k, best[w]);
      last = k;
      if (threadIdx.x == 0) {
        const bool none = undefined || k == 0;
        a.top_ids[(long)t * a.top + j] = none ? -1 : key_id(k);
        a.top_logprobs[(long)t * a.top + j] = undefined ? NAN : k == 0 ? -INFINITY : (key_logit(k) - p.m) - log_s;
      }
    }
  }
}

template <typename E>
int launch(const LogprobArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((logprob_rows_kernel<E>), dim3((unsigned)std::min(a.T, 1 << 20)), dim3(THREADS), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t qmoe_token_logprobs_workspace(int T, int V, int type, int top) {
  (void)T, (void)V, (void)type, (void)top;
  return 0;
}

int qmoe_token_logprobs(const void* logits, long ld, int type, const void* tokens, int m, const void* allowed,
                        long ld_allowed, int T, int V, void* logprobs, void* entropy, int top, void* top_ids,
                        void* top_logprobs, void* workspace, size_t workspace_bytes, void* stream) {
  if (T < 0 || V < 1 || V > (1 << 30) || m < 0 || top < 0 || top > TOP_MAX || ld < 0 || (allowed && ld_allowed < 0)) return QMOE_EINVAL;
  if (T == 0) return QMOE_OK;
  if (!logits || !entropy || (m && (!tokens || !logprobs)) || (top && (!top_ids || !top_logprobs))) return QMOE_EINVAL;
  const size_t need = qmoe_token_logprobs_workspace(T, V, type, top);
  if (need && (!workspace || workspace_bytes < need)) return QMOE_EWORKSPACE;
  LogprobArgs a = {};
  a.logits = logits, a.ld = ld, a.tokens = (const int64_t*)tokens, a.m = m;
  a.allowed = (const uint8_t*)allowed, a.lda = ld_allowed, a.T = T, a.V = V;
  a.logprobs = (float*)logprobs, a.entropy = (float*)entropy;
  a.top = top, a.top_ids = (int64_t*)top_ids, a.top_logprobs = (float*)top_logprobs;
  if (type == QMOE_BF16) return launch<ElemBF16>(a, (hipStream_t)stream);
  if (type == QMOE_F16) return launch<ElemF16>(a, (hipStream_t)stream);
  if (type == QMOE_F32) return launch<ElemF32>(a, (hipStream_t)stream);
  return QMOE_EINVAL;
}

}  // extern "C"
