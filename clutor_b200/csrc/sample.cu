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

constexpr int CL = 8;                        // CTAs of a cluster: one row
constexpr int ST = 512, SW = ST / 32;        // threads and warps of a CTA
constexpr int NB = 1024;                     // bins of a histogram
constexpr int CAP = 512;                     // tokens of one bin that are ordered directly
constexpr int SAMPLE_MAX_VOCAB = 1 << 18;
constexpr double UNIT = 17592186044416.0;    // 2^44
constexpr float BINS_PER_NAT = 32.f;         // the first histogram's bins cover 32 e-foldings: lighter weights are below 2^-44

using u64 = unsigned long long;

// A logit as an unsigned integer in the same order; NaN as -infinity.
CLB_DEV uint32_t key_of(float x) {
  if (x != x) x = -INFINITY;
  if (x == 0.f) x = 0.f;   // -0 is 0
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
CLB_DEV float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// ---- the cluster -----------------------------------------------------------------------------------------------------------
CLB_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
CLB_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
CLB_DEV uint32_t remote(const void *p, uint32_t rank) {   // p's counterpart in another CTA of the cluster
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  return a;
}
CLB_DEV u64 remote_u64(const u64 *p, uint32_t rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}
CLB_DEV uint32_t remote_u32(const uint32_t *p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}

// A place in the order (logit descending, id ascending): what it keeps is the prefix that ends there.
struct Limit {
  uint32_t key;
  uint32_t id;
  CLB_DEV bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= id); }
};

struct Shared {
  u64 sum[NB];          // a histogram's values
  uint32_t cnt[NB];     // and counts
  u64 list[CAP];        // this CTA's tokens of a bin: key, complement of the id
  u64 all[CAP];         // every CTA's
  u64 part[SW + 1];
  u64 mine[4];          // what this CTA tells the others
  u64 found[4];         // what a search found, for the CTA's threads
  uint32_t n_list;
  double exp2_64[64];   // 2^(i / 64)
};

// One row's slice in this CTA, and what is known of the row.
struct Row {
  Shared *sh;
  const uint32_t *key;   // [n] keys of tokens [base, base + n)
  uint32_t n, base, rank, per_thread;
  float top, inv_f;      // the largest logit; 1 / temperature
  double scale;          // log2(e) / temperature
  uint32_t top_key;

  // exp((x - top) / temperature): 2^y with y = n / 64 + r, 2^(n/64) from a table and 2^r by its series (|r| <= 1 / 128: the
  // first term left out is below 4e-17), the table-driven method of Tang (1989).
  CLB_DEV double weight(uint32_t k) const;
  CLB_DEV u64 mass(uint32_t k) const;
  // (top - x) / temperature in bins: equal or larger for smaller logits, so a bin holds one run of the order.
  CLB_DEV uint32_t bin(uint32_t k) const {
    if (k == top_key) return 0;
    const float d = __fmul_rn(__fsub_rn(top, logit_of(k)), inv_f) * BINS_PER_NAT;   // NaN for infinity x 0
    return d < static_cast<float>(NB - 1) ? static_cast<uint32_t>(d) : static_cast<uint32_t>(NB - 1);
  }
};

__device__ const double EXP2_64[64] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284, 1.0442737824274138,
    1.0556451783605572, 1.0671404006768237, 1.0787607977571199, 1.0905077326652577, 1.102382583307841,
    1.1143867425958924, 1.1265216186082418, 1.1387886347566916, 1.1511892299529827, 1.1637248587775775,
    1.1763969916502812, 1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783, 1.2968395546510096,
    1.3109612115247644, 1.3252366431597413, 1.339667524053303, 1.3542555469368927, 1.3690024229745905,
    1.383909881963832, 1.3989796725383112, 1.4142135623730951, 1.42961333839197, 1.4451808069770467,
    1.460917794180647, 1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267, 1.6104903319492543,
    1.6280274218573478, 1.645755478153965, 1.6636765803267364, 1.681792830507429, 1.7001063537185235,
    1.718619298122478, 1.7373338352737062, 1.7562521603732995, 1.7753764925265212, 1.7947090750031072,
    1.8142521755003989, 1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951,
};

CLB_DEV double Row::weight(uint32_t k) const {
  if (k == top_key) return 1.0;
  const float x = logit_of(k);
  if (top == INFINITY || x == -INFINITY) return 0.0;
  const double y = (static_cast<double>(x) - static_cast<double>(top)) * scale;
  if (!(y > -1000.0)) return 0.0;
  const double t = y * 64.0 + 6755399441055744.0;   // 1.5 * 2^52: the nearest integer in the low bits
  const int n = __double2loint(t);
  const double r = fma(t - 6755399441055744.0, -1.0 / 64.0, y) * 0.6931471805599453;
  double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  p *= sh->exp2_64[n & 63];
  return __hiloint2double(__double2hiint(p) + (n >> 6) * (1 << 20), __double2loint(p));   // p in [0.99, 2), n >> 6 >= -1001: a normal number
}
CLB_DEV u64 Row::mass(uint32_t k) const { return __double2ull_rn(weight(k) * UNIT); }

// The sum of the threads' values before this thread's, and (total) of all.
CLB_DEV u64 block_scan(Shared *sh, u64 v, u64 &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 u = __shfl_up_sync(FULL_MASK, s, o);
    if (lane >= o) s += u;
  }
  __syncthreads();
  if (lane == 31) sh->part[warp] = s;
  __syncthreads();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < SW; ++w) {
    const u64 u = sh->part[w];
    if (w < warp) before += u;
    total += u;
  }
  return before + s - v;
}
// The CTAs' values v (the same in every thread of a CTA) before this CTA's, and of all.
CLB_DEV u64 cluster_scan(Row &r, u64 v, u64 &total) {
  Shared *sh = r.sh;
  cluster_sync();   // what was exchanged before has been read
  if (threadIdx.x == 0) sh->mine[0] = v;
  cluster_sync();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (uint32_t c = 0; c < CL; ++c) {
    const u64 u = remote_u64(&sh->mine[0], c);
    if (c < r.rank) before += u;
    total += u;
  }
  return before;
}

// The end of the shortest prefix of the order, among the tokens that `among` keeps, whose values (masses, or ones) sum to at
// least `want` -- for masses ceil(share x their total). Histograms over ever finer runs of the order, summed over the cluster
// by every CTA for itself, narrow it to a bin of at most CAP tokens, which are sorted, or to one key, whose tokens count by id.
template <bool MASS>
CLB_DEV Limit prefix(Row &r, const Limit &among, u64 want, double share) {
  Shared *sh = r.sh;
  const int tid = threadIdx.x;
  uint32_t lo = 0, hi = 0, shift = 0;   // the run that a level divides: at level 0 everything, then the keys [lo, hi]
  for (int level = 0;; ++level) {
    auto inside = [&](uint32_t k, uint32_t i) {   // whether a token belongs to the run that this level divides
      if (!among.keeps(k, r.base + i)) return false;
      return level == 0 || (k >= lo && k <= hi);
    };
    auto place = [&](uint32_t k) { return level == 0 ? r.bin(k) : (hi - k) >> shift; };
    for (int b = tid; b < NB; b += ST) { sh->sum[b] = 0; sh->cnt[b] = 0; }
    __syncthreads();
    for (uint32_t i = tid; i < r.n; i += ST) {
      const uint32_t k = r.key[i];
      if (!inside(k, i)) continue;
      const uint32_t b = place(k);
      atomicAdd(&sh->cnt[b], 1u);
      if (MASS) {
        const u64 m = r.mass(k);
        if (m) atomicAdd(&sh->sum[b], m);
      }
    }
    cluster_sync();
    u64 v[NB / ST], mine = 0;
    uint32_t n[NB / ST];
#pragma unroll
    for (int e = 0; e < NB / ST; ++e) {
      const int b = tid * (NB / ST) + e;
      v[e] = 0;
      n[e] = 0;
#pragma unroll
      for (uint32_t c = 0; c < CL; ++c) {
        n[e] += remote_u32(&sh->cnt[b], c);
        if (MASS) v[e] += remote_u64(&sh->sum[b], c);
      }
      if (!MASS) v[e] = n[e];
      mine += v[e];
    }
    u64 total;
    u64 before = block_scan(sh, mine, total);
    if (MASS && level == 0) {
      const double w = ceil(share * static_cast<double>(total));
      want = w >= static_cast<double>(total) ? total : w < 1.0 ? 1ull : static_cast<u64>(w);
    }
#pragma unroll
    for (int e = 0; e < NB / ST; ++e) {
      if (before < want && before + v[e] >= want) {
        sh->found[0] = tid * (NB / ST) + e;
        sh->found[1] = before;
        sh->found[2] = n[e];
      }
      before += v[e];
    }
    if (tid == 0) sh->n_list = 0;
    __syncthreads();
    const uint32_t b = static_cast<uint32_t>(sh->found[0]), count = static_cast<uint32_t>(sh->found[2]);
    want -= sh->found[1];
    if (count <= CAP) {   // few: every CTA lists its own, then sorts everybody's
      for (uint32_t i = tid; i < r.n; i += ST) {
        const uint32_t k = r.key[i];
        if (inside(k, i) && place(k) == b) sh->list[atomicAdd(&sh->n_list, 1u)] = (static_cast<u64>(k) << 32) | (0xffffffffu - (r.base + i));
      }
      cluster_sync();
      uint32_t at = 0;
      for (uint32_t c = 0; c < CL; ++c) {
        const uint32_t m = remote_u32(&sh->n_list, c);
        if (tid >= at && tid < at + m) sh->all[tid] = remote_u64(&sh->list[tid - at], c);
        at += m;
      }
      __syncthreads();
      cluster_sync();   // the lists and histograms have been read
      u64 x = static_cast<uint32_t>(tid) < count ? sh->all[tid] : 0;   // descending; 0 sorts last
      int size = 1;
      while (size < static_cast<int>(count)) size <<= 1;
      for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
          u64 y;
          if (j >= 32) {
            __syncthreads();
            sh->all[tid] = x;
            __syncthreads();
            y = sh->all[tid ^ j];
          } else {
            y = __shfl_xor_sync(FULL_MASK, x, j);
          }
          const bool first = (tid & j) == 0, down = (tid & k) == 0;   // down: the larger first
          x = (x > y) == (first == down) ? x : y;
        }
      const uint32_t k = static_cast<uint32_t>(x >> 32);
      const u64 val = static_cast<uint32_t>(tid) < count ? (MASS ? r.mass(k) : 1ull) : 0ull;
      const u64 s = block_scan(sh, val, total);
      if (s < want && s + val >= want) sh->found[3] = x;
      __syncthreads();
      const u64 f = sh->found[3];
      return Limit{static_cast<uint32_t>(f >> 32), 0xffffffffu - static_cast<uint32_t>(f)};
    }
    // the keys of that bin, and their range over the cluster
    uint32_t kmin = 0xffffffffu, kmax = 0;
    for (uint32_t i = tid; i < r.n; i += ST) {
      const uint32_t k = r.key[i];
      if (inside(k, i) && place(k) == b) { kmin = min(kmin, k); kmax = max(kmax, k); }
    }
    kmin = __reduce_min_sync(FULL_MASK, kmin);
    kmax = __reduce_max_sync(FULL_MASK, kmax);
    __syncthreads();
    if ((tid & 31) == 0) sh->part[tid >> 5] = (static_cast<u64>(kmax) << 32) | kmin;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < SW; ++w) {
        kmin = min(kmin, static_cast<uint32_t>(sh->part[w]));
        kmax = max(kmax, static_cast<uint32_t>(sh->part[w] >> 32));
      }
      sh->mine[1] = (static_cast<u64>(kmax) << 32) | kmin;
    }
    cluster_sync();
    lo = 0xffffffffu;
    hi = 0;
    for (uint32_t c = 0; c < CL; ++c) {
      const u64 m = remote_u64(&sh->mine[1], c);
      lo = min(lo, static_cast<uint32_t>(m));
      hi = max(hi, static_cast<uint32_t>(m >> 32));
    }
    if (lo == hi) {   // one key: the q-th of its tokens by id
      const u64 one = MASS ? r.mass(lo) : 1ull, q = one ? (want + one - 1) / one : 1;
      u64 c = 0, t;
      const uint32_t i0 = tid * r.per_thread, i1 = min(i0 + r.per_thread, r.n);
      for (uint32_t i = i0; i < i1; ++i) c += r.key[i] == lo && among.keeps(lo, r.base + i);
      u64 s = block_scan(sh, c, t);
      u64 cl_total;
      s += cluster_scan(r, t, cl_total);
      if (tid == 0) sh->mine[2] = 0;
      __syncthreads();
      if (s < q && s + c >= q)
        for (uint32_t i = i0; i < i1; ++i)
          if (r.key[i] == lo && among.keeps(lo, r.base + i) && ++s == q) sh->mine[2] = r.base + i + 1ull;
      cluster_sync();
      u64 id = 0;
      for (uint32_t d = 0; d < CL; ++d) id = max(id, remote_u64(&sh->mine[2], d));
      cluster_sync();
      return Limit{lo, static_cast<uint32_t>(id - 1)};
    }
    const int bits = 32 - __clz(hi - lo);
    shift = bits > 10 ? bits - 10 : 0;
    cluster_sync();   // the ranges and the histograms have been read
  }
}

// One row by one cluster: its keys lie in the CTAs' shared memory, a slice each, and are read from memory once.
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(ST, 2) sample_kernel(const clb200_sampling s, const uint32_t slice) {
  extern __shared__ __align__(16) uint8_t sm[];
  Shared *sh = reinterpret_cast<Shared *>(sm);
  uint32_t *key = reinterpret_cast<uint32_t *>(sh + 1);
  const int row = blockIdx.x / CL, tid = threadIdx.x;
  Row r;
  r.sh = sh;
  r.key = key;
  r.rank = cluster_rank();
  r.base = r.rank * slice;
  r.n = r.base < static_cast<uint32_t>(s.vocab) ? min(slice, static_cast<uint32_t>(s.vocab) - r.base) : 0;
  r.per_thread = ((slice + ST - 1) / ST) | 1;   // odd: a warp's threads read different banks
  if (tid < 64) sh->exp2_64[tid] = EXP2_64[tid];
  // the keys, and the largest with the lowest id
  u64 best = 0;
  const int64_t at = row * s.stride + r.base;
#pragma unroll 8
  for (uint32_t i = tid; i < r.n; i += ST) {
    const float x = s.type == T_F32 ? static_cast<const float *>(s.logits)[at + i]
                    : s.type == T_F16 ? to_f32(static_cast<const __half *>(s.logits)[at + i]) : to_f32(static_cast<const __nv_bfloat16 *>(s.logits)[at + i]);
    const uint32_t k = key_of(x);
    key[i] = k;
    best = max(best, (static_cast<u64>(k) << 32) | (0xffffffffu - (r.base + i)));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(FULL_MASK, best, o));
  if ((tid & 31) == 0) sh->part[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < SW; ++w) best = max(best, sh->part[w]);
    sh->mine[3] = best;
  }
  cluster_sync();
  best = 0;
  for (uint32_t c = 0; c < CL; ++c) best = max(best, remote_u64(&sh->mine[3], c));
  r.top_key = static_cast<uint32_t>(best >> 32);
  r.top = logit_of(r.top_key);
  const float t = s.temperature ? s.temperature[row] : 1.f;
  if (r.top == -INFINITY || !(t > 0.f)) {
    if (r.rank == 0 && tid == 0) {
      s.token[row] = r.top == -INFINITY ? -1 : static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
      if (s.prob) s.prob[row] = r.top == -INFINITY ? 0.f : 1.f;
    }
    cluster_sync();   // the others may still be reading this CTA's shared memory
    return;
  }
  r.inv_f = 1.0f / t;
  r.scale = 1.4426950408889634 / static_cast<double>(t);
  const int k = s.top_k ? s.top_k[row] : 0;
  const float share = s.top_p ? s.top_p[row] : 1.f, least = s.min_p ? s.min_p[row] : 0.f;
  const double min_w = least > 0.f ? fmin(static_cast<double>(least), 1.0) : 0.0;
  Limit lim{0, 0xffffffffu};
  if (k > 0 && k < s.vocab) lim = prefix<false>(r, lim, static_cast<u64>(k), 0.0);
  if (share < 1.f) lim = prefix<true>(r, lim, 0, static_cast<double>(share));
  auto kept = [&](uint32_t q, uint32_t i) -> u64 {
    if (!lim.keeps(q, r.base + i)) return 0;
    const double w = r.weight(q);
    return w >= min_w ? __double2ull_rn(w * UNIT) : 0ull;
  };
  // the kept masses by id: a thread's tokens, the threads before it, the CTAs before its own
  u64 mine = 0, cta_total, total;
  const uint32_t i0 = tid * r.per_thread, i1 = min(i0 + r.per_thread, r.n);
  for (uint32_t i = i0; i < i1; ++i) mine += kept(key[i], i);
  u64 before = block_scan(sh, mine, cta_total);
  before += cluster_scan(r, cta_total, total);
  const double u = fmin(fmax(static_cast<double>(s.u[row]), 0.0), 1.0);   // a NaN counts as 0
  const u64 want = min(static_cast<u64>(u * static_cast<double>(total)), total - 1);
  if (before <= want && want < before + mine) {
    for (uint32_t i = i0; i < i1; ++i) {
      before += kept(key[i], i);
      if (before > want) {
        s.token[row] = static_cast<int>(r.base + i);
        if (s.prob) s.prob[row] = static_cast<float>(r.weight(key[i]) / (static_cast<double>(total) * (1.0 / UNIT)));
        break;
      }
    }
  }
  cluster_sync();
}

int check(const clb200_sampling *s, char *err, size_t errlen) {
  if (!s) { errf(err, errlen, "no arguments"); return 1; }
  if (s->rows < 0 || s->rows > (1 << 24) || s->vocab < 1 || s->vocab > SAMPLE_MAX_VOCAB) {
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
  const uint32_t slice = (static_cast<uint32_t>(s->vocab) + CL - 1) / CL;
  const size_t smem = sizeof(Shared) + static_cast<size_t>(slice) * 4;
  static bool done[64] = {};
  if (c->device >= 64 || !done[c->device]) {
    CUDA_OR(cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(Shared) + SAMPLE_MAX_VOCAB / CL * 4)),
            "kernel attribute");
    if (c->device < 64) done[c->device] = true;
  }
  sample_kernel<<<static_cast<unsigned>(s->rows) * CL, ST, smem, stream ? static_cast<cudaStream_t>(stream) : c->stream>>>(*s, slice);
  CUDA_OR(cudaGetLastError(), "launching the sampling");
  return 0;
}
