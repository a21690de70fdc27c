// clb200_sample: the choice of a token from logits by temperature, top-k, top-p and min-p, from given random numbers.
//
// Every filter keeps a prefix of the tokens ordered by (logit descending, id ascending), so a filter is a pair (key, id): a
// token is kept when its key is larger, or equal with an id at most that one. Keys are the logits' bits made monotone.
// Weights are 64-bit integers, w = round(exp((x - M) / temperature) * 2^44): at most 2^18 of at most 2^44 fit 62 bits, and
// integer sums do not depend on their order.
#include <algorithm>

#include "ctx.cuh"
#include "serve.cuh"

namespace clb {
namespace {

constexpr int ST = 1024, SW = ST / 32;
constexpr int SAMPLE_MAX_VOCAB = 1 << 18;
constexpr double UNIT = 17592186044416.0;   // 2^44

// A logit as an unsigned integer in the same order; NaN as -infinity.
CLB_DEV uint32_t key_of(float x) {
  if (x != x) x = -INFINITY;
  if (x == 0.f) x = 0.f;   // -0 is 0
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
CLB_DEV float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

struct Pick {
  const clb200_sampling *s;
  const void *row;
  int vocab;
  uint32_t type;
  float top;
  double inv_t;
  CLB_DEV float logit(int i) const {
    if (type == T_F32) return static_cast<const float *>(row)[i];
    if (type == T_F16) return to_f32(static_cast<const __half *>(row)[i]);
    return to_f32(static_cast<const __nv_bfloat16 *>(row)[i]);
  }
  CLB_DEV double weight(uint32_t key) const {
    const float x = logit_of(key);
    if (x == top) return 1.0;   // also where both are +infinity
    if (top == INFINITY || x == -INFINITY) return 0.0;
    return exp((static_cast<double>(x) - static_cast<double>(top)) * inv_t);
  }
  CLB_DEV unsigned long long mass(uint32_t key) const { return static_cast<unsigned long long>(weight(key) * UNIT + 0.5); }
};

// The block's sum of v, for every thread.
CLB_DEV unsigned long long block_sum(unsigned long long v) {
  __shared__ unsigned long long part[SW];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned long long t = 0;
  for (int w = 0; w < SW; ++w) t += part[w];
  return t;
}

template <typename F>
CLB_DEV unsigned long long row_sum(const Pick &p, F f) {
  unsigned long long v = 0;
  for (int i = threadIdx.x; i < p.vocab; i += ST) v += f(key_of(p.logit(i)), i);
  return block_sum(v);
}

struct Limit {
  uint32_t key;
  int id;
  CLB_DEV bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= id); }
};

// The shortest prefix of the order whose values sum to at least want (> 0); value(key, id) is the same for equal keys.
template <typename F>
CLB_DEV Limit prefix(const Pick &p, unsigned long long want, F value) {
  uint32_t key = 0;
  for (int b = 31; b >= 0; --b) {
    const uint32_t c = key | (1u << b);
    if (row_sum(p, [&](uint32_t k, int i) { return k >= c ? value(k, i) : 0ull; }) >= want) key = c;
  }
  const unsigned long long above = row_sum(p, [&](uint32_t k, int i) { return k > key ? value(k, i) : 0ull; });
  int lo = 0, hi = p.vocab - 1;   // the lowest id at which the tokens of this key, ids ascending, make up the rest
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (above + row_sum(p, [&](uint32_t k, int i) { return k == key && i <= mid ? value(k, i) : 0ull; }) >= want) hi = mid;
    else lo = mid + 1;
  }
  return Limit{key, lo};
}

__global__ void __launch_bounds__(ST) sample_plain_kernel(const clb200_sampling s) {
  const int r = blockIdx.x;
  const size_t size = s.type == T_F32 ? 4 : 2;
  Pick p{&s, static_cast<const uint8_t *>(s.logits) + r * s.stride * size, s.vocab, s.type, 0.f, 1.0};
  __shared__ unsigned long long best;
  if (threadIdx.x == 0) best = 0;
  __syncthreads();
  unsigned long long b = 0;
  for (int i = threadIdx.x; i < p.vocab; i += ST) {
    const unsigned long long v = (static_cast<unsigned long long>(key_of(p.logit(i))) << 32) | (0xffffffffu - i);
    b = v > b ? v : b;
  }
  atomicMax(&best, b);
  __syncthreads();
  const uint32_t top_key = static_cast<uint32_t>(best >> 32);
  const int top_id = static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
  p.top = logit_of(top_key);
  const float t = s.temperature ? s.temperature[r] : 1.f;
  if (p.top == -INFINITY || !(t > 0.f)) {
    if (threadIdx.x == 0) {
      s.token[r] = p.top == -INFINITY ? -1 : top_id;
      if (s.prob) s.prob[r] = p.top == -INFINITY ? 0.f : 1.f;
    }
    return;
  }
  p.inv_t = 1.0 / static_cast<double>(t);
  const int k = s.top_k ? s.top_k[r] : 0;
  const float pp = s.top_p ? s.top_p[r] : 1.f;
  const float mf = s.min_p ? s.min_p[r] : 0.f;
  const double mp = mf > 0.f ? fmin(static_cast<double>(mf), 1.0) : 0.0;
  Limit top_k{0, p.vocab}, top_p{0, p.vocab};
  if (k > 0 && k < p.vocab) top_k = prefix(p, static_cast<unsigned long long>(k), [&](uint32_t, int) { return 1ull; });
  if (pp < 1.f) {
    const unsigned long long total = row_sum(p, [&](uint32_t q, int i) { return top_k.keeps(q, i) ? p.mass(q) : 0ull; });
    const double want = fmax(ceil(static_cast<double>(pp) * static_cast<double>(total)), 1.0);
    const unsigned long long w = min(static_cast<unsigned long long>(want), total);
    top_p = prefix(p, w, [&](uint32_t q, int) { return p.mass(q); });
  }
  auto kept = [&](uint32_t q, int i) -> unsigned long long {
    return top_k.keeps(q, i) && top_p.keeps(q, i) && p.weight(q) >= mp ? p.mass(q) : 0ull;
  };
  const unsigned long long total = row_sum(p, kept);
  const double u = fmin(fmax(static_cast<double>(s.u[r]), 0.0), 1.0);   // a NaN counts as 0
  const unsigned long long want = min(static_cast<unsigned long long>(u * static_cast<double>(total)), total - 1);
  int lo = 0, hi = p.vocab - 1;   // the lowest id at which the running sum exceeds want
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (row_sum(p, [&](uint32_t q, int i) { return i <= mid ? kept(q, i) : 0ull; }) > want) hi = mid;
    else lo = mid + 1;
  }
  if (threadIdx.x == 0) {
    s.token[r] = lo;
    if (s.prob) s.prob[r] = static_cast<float>(p.weight(key_of(p.logit(lo))) / (static_cast<double>(total) * (1.0 / UNIT)));
  }
}

int check(const clb200_sampling *s, char *err, size_t errlen) {
  if (!s) { errf(err, errlen, "no arguments"); return 1; }
  if (s->rows < 0 || s->vocab < 1 || s->vocab > SAMPLE_MAX_VOCAB) {
    errf(err, errlen, "%d rows of %d logits: takes 1 to %d logits a row", s->rows, s->vocab, SAMPLE_MAX_VOCAB);
    return 1;
  }
  if (s->type != T_F32 && s->type != T_F16 && s->type != T_BF16) { errf(err, errlen, "logits are %s: F32, F16 or BF16", type_name(s->type)); return 1; }
  if (!s->logits || !s->u || !s->token) { errf(err, errlen, "a buffer is missing"); return 1; }
  if (s->rows > 1 && s->stride < s->vocab) { errf(err, errlen, "rows %lld elements apart do not hold %d logits", (long long)s->stride, s->vocab); return 1; }
  if (reinterpret_cast<uintptr_t>(s->logits) % (s->type == T_F32 ? 4 : 2)) { errf(err, errlen, "the logits do not start on a boundary of their type"); return 1; }
  return 0;
}

}  // namespace
}  // namespace clb

using namespace clb;

extern "C" int clb200_sample(clb200_ctx *c, const clb200_sampling *s, void *stream, char *err, size_t errlen) {
  if (check(s, err, errlen)) return 1;
  if (!c) { errf(err, errlen, "no context"); return 1; }
  if (s->rows == 0) return 0;
  const OnDevice on(c->device);
  sample_plain_kernel<<<s->rows, ST, 0, stream ? static_cast<cudaStream_t>(stream) : c->stream>>>(*s);
  CUDA_OR(cudaGetLastError(), "launching the sampling");
  return 0;
}
