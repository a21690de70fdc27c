// clb200_sample: the choice of a token from logits by temperature, top-k, top-p and min-p, from given random numbers.
//
// Every filter keeps a prefix of the tokens ordered by (logit descending, id ascending), so a filter is a pair (key, id): a
// token is kept when its key is larger, or equal with an id at most that one. A key is a logit's bits made monotone.
// Weights are 64-bit integers, w = round(exp((x - M) / temperature) * 2^44): at most 2^18 of at most 2^44 fit 62 bits, and
// integer sums do not depend on their order.
//
// A row's bytes are read once, and that would take 6 us for 64 rows of 151936; what it does take (57) is a chain: the largest, a
// histogram over runs of the order (bins of 1/64 in the exponent), the bin that holds the border, that bin's tokens sorted, and for
// a broad nucleus the weight of every token, twice, in double precision (256 rows of 50304: 84 us; the issue slots are 83 % taken,
// the ALU pipe 54 %, the double pipe 24 %). So the logits stay in shared memory, phases are few, a small set of candidates is sorted
// once and answers everything, and rows are spread over CTAs by the rule at the launch.
#include <algorithm>

#include "ctx.cuh"
#include "serve.cuh"

namespace clb {
namespace {

constexpr int NB = 2048;                     // bins of a histogram
constexpr int CAP = 512;                     // tokens that are sorted directly, at most (a thread each)
constexpr int E = 4;                         // tokens a thread weighs at once
constexpr int SAMPLE_MAX_VOCAB = 1 << 18;
constexpr double UNIT = 17592186044416.0;    // 2^44
constexpr float BINS_PER_NAT = 64.f;         // the first histogram's bins cover 32 e-foldings: lighter weights are below 2^-44

using u64 = unsigned long long;

// A logit (not NaN, not -0) as an unsigned integer in the same order.
CLB_DEV uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ (static_cast<uint32_t>(static_cast<int>(b) >> 31) | 0x80000000u);
}
CLB_DEV float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
constexpr uint32_t KEY_LOWEST = 0x007fffffu;   // of -infinity

// ---- the cluster: CL CTAs, one row -----------------------------------------------------------------------------------------
template <int CL>
CLB_DEV uint32_t cluster_rank() {
  uint32_t r = 0;
  if constexpr (CL > 1) asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
template <int CL>
CLB_DEV void cluster_sync() {
  if constexpr (CL > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();
}
// A word of another CTA's shared memory, at the place that p has in this one's.
template <int CL>
CLB_DEV u64 remote(const u64 *p, uint32_t rank) {
  if constexpr (CL == 1) return *p;
  u64 v;
  asm volatile("{\n .reg .u32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.u64 %0, [a];\n}\n" : "=l"(v) : "r"(smem_addr(p)), "r"(rank) : "memory");
  return v;
}
template <int CL>
CLB_DEV uint32_t remote(const uint32_t *p, uint32_t rank) {
  if constexpr (CL == 1) return *p;
  uint32_t v;
  asm volatile("{\n .reg .u32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.u32 %0, [a];\n}\n" : "=r"(v) : "r"(smem_addr(p)), "r"(rank) : "memory");
  return v;
}

// A place in the order (logit descending, id ascending): what it keeps is the prefix that ends there.
struct Limit {
  uint32_t key;
  uint32_t id;
  CLB_DEV bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= id); }
  CLB_DEV bool all() const { return key <= KEY_LOWEST && id == 0xffffffffu; }
};
CLB_DEV u64 token_word(uint32_t key, uint32_t id) { return (static_cast<u64>(key) << 32) | (0xffffffffu - id); }   // larger first in the order

struct Shared {
  uint32_t lo[NB], hi[NB];   // a histogram: counts in lo, or the halves of 64-bit sums
  u64 coarse[32];            // the sums of NB / 32 bins each
  u64 list[CAP];             // this CTA's tokens of a search, as token_word
  u64 all[CAP];              // every CTA's
  u64 part[32];
  u64 mine[4];               // what this CTA tells the others
  u64 found[7];              // what a search found, for the CTA's threads
  uint32_t n_list, n_above;
  double exp2_128[128];      // 2^(i / 128), i << 13 taken from the upper word
};
static_assert(sizeof(Shared) % 16 == 0, "the logits follow on a 16-byte boundary");

__device__ const double EXP2_128[128] = {
    1.0, 1.0054299011128027, 1.0108892860517005, 1.016378314910953, 1.0218971486541166,
    1.0274459491187637, 1.0330248790212284, 1.0386341019613787, 1.0442737824274138, 1.0499440858006872,
    1.0556451783605572, 1.061377227289262, 1.0671404006768237, 1.0729348675259756, 1.0787607977571199,
    1.0846183622133092, 1.0905077326652577, 1.0964290818163769, 1.102382583307841, 1.1083684117236787,
    1.1143867425958924, 1.1204377524096067, 1.1265216186082418, 1.1326385195987192, 1.1387886347566916,
    1.1449721444318042, 1.1511892299529827, 1.1574400736337511, 1.1637248587775775, 1.1700437696832502,
    1.1763969916502812, 1.182784710984341, 1.189207115002721, 1.1956643920398273, 1.202156731452703,
    1.2086843236265816, 1.215247359980469, 1.2218460329727576, 1.22848053610687, 1.2351510639369334,
    1.241857812073484, 1.2486009771892048, 1.255380757024691, 1.2621973503942507, 1.2690509571917332,
    1.275941778396392, 1.2828700160787783, 1.2898358734066657, 1.2968395546510096, 1.3038812651919358,
    1.3109612115247644, 1.318079601266064, 1.3252366431597413, 1.3324325470831615, 1.339667524053303,
    1.3469417862329458, 1.3542555469368927, 1.3616090206382248, 1.3690024229745905, 1.3764359707545302,
    1.383909881963832, 1.3914243757719262, 1.3989796725383112, 1.4065759938190154, 1.4142135623730951,
    1.4218926021691656, 1.42961333839197, 1.4373759974489824, 1.4451808069770467, 1.4530279958490526,
    1.460917794180647, 1.4688504333369818, 1.4768261459394993, 1.4848451658727524, 1.4929077282912648,
    1.5010140696264256, 1.5091644275934228, 1.5173590411982147, 1.5255981507445384, 1.533881997840956,
    1.5422108254079407, 1.550584877685, 1.559004400237837, 1.567469639965553, 1.5759808451078865,
    1.5845382652524937, 1.593142151342267, 1.6017927556826934, 1.6104903319492543, 1.6192351351948637,
    1.6280274218573478, 1.6368674497669644, 1.645755478153965, 1.6546917676561943, 1.6636765803267364,
    1.6727101796415966, 1.681792830507429, 1.6909247992693053, 1.7001063537185235, 1.709337763100463,
    1.718619298122478, 1.7279512309618377, 1.7373338352737062, 1.746767386199169, 1.7562521603732995,
    1.7657884359332727, 1.7753764925265212, 1.785016611318935, 1.7947090750031072, 1.804454167806624,
    1.8142521755003989, 1.8241033854070534, 1.8340080864093424, 1.843966568958626, 1.8539791250833855,
    1.864046048397789, 1.8741676341103, 1.8843441790323345, 1.8945759815869656, 1.9048633418176741,
    1.9152065613971474, 1.925605943636125, 1.9360617934922943, 1.9465744175792332, 1.9571441241754002,
    1.9677712232331759, 1.978456026387951, 1.9891988469672663,
};

constexpr int SAMPLE_SMEM = 227 * 1024;
constexpr uint32_t MAX_SLICE = (SAMPLE_SMEM - sizeof(Shared)) / 4 - 3;

// One row's slice in this CTA, and what is known of the row.
// w (at most 1) in units of 2^-44, rounded to the nearest: the sum with 2^52 has it in its low bits.
CLB_DEV u64 units(double w) { return static_cast<u64>(__double_as_longlong(fma(w, UNIT, 4503599627370496.0))) & 0xfffffffffffffull; }

CLB_DEV float cleaned(float v) { return fmaxf(v, -INFINITY) + 0.f; }   // NaN as -infinity, -0 as 0

struct Row {
  Shared *sh;
  float *x;              // [n] logits of tokens [base, base + n): NaN as -infinity, no -0
  uint32_t n, base, rank, per_thread;
  float top, half_top, inv_f;   // the largest logit (finite), half of it; 1 / temperature
  float heat, floor;     // the temperature; logits up to this weigh nothing
  double top_d, scale;   // log2(e) / temperature

  // (top - x) / (2 temperature): halved so that it does not overflow; NaN for infinity x 0.
  CLB_DEV float distance(float v) const { return __fmul_rn(fmaf(v, -0.5f, half_top), inv_f); }
  // exp((x - top) / temperature) = 2^y with y = n / 128 + r: 2^(n/128) from a table and 2^r by its series (|r| <= 1 / 256: the
  // first term left out is below 1.3e-15), the table-driven method of Tang (1989). COUNT at once and without branches: one alone is
  // a chain of a dozen dependent double-precision operations. What bounds them is the ALU pipe (compares, selects, logic), which
  // takes a warp's instruction in two cycles: so the table's entries have i << 13 taken from their upper words, and n << 13 added
  // to one gives 2^(n/128) in a single multiply-add.
  template <int COUNT>
  CLB_DEV void weights(const float (&v)[COUNT], double (&w)[COUNT]) const {
    double y[COUNT], t[COUNT];
#pragma unroll
    for (int e = 0; e < COUNT; ++e) y[e] = (static_cast<double>(v[e] > floor ? v[e] : top) - top_d) * scale;
#pragma unroll
    for (int e = 0; e < COUNT; ++e) t[e] = fma(y[e], 128.0, 6755399441055744.0);   // 1.5 * 2^52: the nearest integer in the low bits
#pragma unroll
    for (int e = 0; e < COUNT; ++e) y[e] = fma(t[e] - 6755399441055744.0, -1.0 / 128.0, y[e]);
#pragma unroll
    for (int e = 0; e < COUNT; ++e) w[e] = fma(y[e], 0.009618129107628477, 0.05550410866482158);   // ln(2)^4 / 24, ln(2)^3 / 6
#pragma unroll
    for (int e = 0; e < COUNT; ++e) w[e] = fma(w[e], y[e], 0.2402265069591007);
#pragma unroll
    for (int e = 0; e < COUNT; ++e) w[e] = fma(w[e], y[e], 0.6931471805599453);
#pragma unroll
    for (int e = 0; e < COUNT; ++e) {
      const int n = __double2loint(t[e]);
      const double p = sh->exp2_128[n & 127];
      // what weighs nothing keeps the lower word alone: below 2^-1022
      w[e] = fma(w[e], y[e], 1.0) * __hiloint2double(v[e] > floor ? n * 8192 + __double2hiint(p) : 0, __double2loint(p));
    }
  }
  CLB_DEV double weight(float v) const {
    const float q[1] = {v};
    double w[1];
    weights(q, w);
    return w[0];
  }
  CLB_DEV u64 mass(uint32_t k) const { return units(weight(logit_of(k))); }
  // (top - x) / temperature in bins: equal or larger for smaller logits, so a bin holds one run of the order.
  CLB_DEV uint32_t bin(float v) const {
    const float d = __fmul_rn(distance(v), 2.f * BINS_PER_NAT);
    return static_cast<uint32_t>(fminf(d, static_cast<float>(NB - 1)));
  }
};

// Sums over a warp's lanes up to and with each.
CLB_DEV u64 warp_scan(u64 s) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 u = __shfl_up_sync(FULL_MASK, s, o);
    if (lane >= o) s += u;
  }
  return s;
}
// The sum of the threads' values before this thread's, and (total) of all.
template <int ST>
CLB_DEV u64 block_scan(Shared *sh, u64 v, u64 &total) {
  constexpr int SW = ST / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64 s = warp_scan(v);
  __syncthreads();
  if (lane == 31) sh->part[warp] = s;
  __syncthreads();
  const u64 w = warp_scan(lane < SW ? sh->part[lane] : 0);
  total = __shfl_sync(FULL_MASK, w, 31);
  const u64 before = __shfl_sync(FULL_MASK, w, max(warp - 1, 0));
  return (warp ? before : 0) + s - v;
}
// The CTAs' values v (the same in every thread of a CTA) before this CTA's, and of all.
template <int CL>
CLB_DEV u64 cluster_scan(Row &r, u64 v, u64 &total) {
  if constexpr (CL == 1) {
    total = v;
    return 0;
  }
  cluster_sync<CL>();   // what was exchanged before has been read
  if (threadIdx.x == 0) r.sh->mine[0] = v;
  cluster_sync<CL>();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (uint32_t c = 0; c < CL; ++c) {
    const u64 u = remote<CL>(&r.sh->mine[0], c);
    if (c < r.rank) before += u;
    total += u;
  }
  return before;
}
// Threads 0 .. n - 1 (n at most MOST) hold words, the others 0; sorts them descending (bitonic).
template <int MOST>
CLB_DEV u64 sort_words(Shared *sh, u64 x, int n) {
  const int tid = threadIdx.x;
  int size = 1;
  while (size < n) size <<= 1;
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      u64 y;
      if (j >= 32) {
        if (tid < MOST) {   // whole warps
          asm volatile("bar.sync 1, %0;" ::"n"(MOST) : "memory");
          sh->all[tid] = x;
          asm volatile("bar.sync 1, %0;" ::"n"(MOST) : "memory");
          y = sh->all[tid ^ j];
        } else {
          y = 0;
        }
      } else {
        y = __shfl_xor_sync(FULL_MASK, x, j);
      }
      const bool first = (tid & j) == 0, down = (tid & k) == 0;   // down: the larger first
      x = (x > y) == (first == down) ? x : y;
    }
  return tid < n ? x : 0;
}
// Every CTA's listed tokens, to every CTA: thread i gets the i-th.
template <int CL>
CLB_DEV u64 gather(Row &r, uint32_t &n) {
  Shared *sh = r.sh;
  const uint32_t tid = threadIdx.x;
  uint32_t m[CL], at = 0;
#pragma unroll
  for (uint32_t c = 0; c < CL; ++c) m[c] = remote<CL>(&sh->n_list, c);
  u64 x = 0;
#pragma unroll
  for (uint32_t c = 0; c < CL; ++c) {
    if (tid >= at && tid < at + m[c]) x = remote<CL>(&sh->list[tid - at], c);
    at += m[c];
  }
  n = at;
  return x;
}

// A search's outcome: the end of the prefix, or, `few`, all the tokens of the prefix and of the bin that it ends in, sorted (thread
// i the i-th of n); and the total mass of the tokens searched (masses only).
struct Found {
  Limit lim;
  bool few;
  u64 word;
  uint32_t n;
  u64 total;
};

// The end of the shortest prefix of the order, among the tokens that `among` keeps, whose values (masses, or ones) sum to at
// least `want` -- for masses ceil(share x their total). Histograms over ever finer runs of the order, summed over the cluster,
// narrow it to a bin of at most MOST tokens, which are sorted, or to one key, whose tokens count by id. Where the tokens before
// the bin are few as well (allow_few) they are all listed and left to the caller. largest: each thread's largest logit, for a
// first try on counts: the want-th largest of those is a lower bound of the want-th largest of all, so the tokens from its bin on
// are listed without a histogram of all of them.
template <int CL, int ST, bool MASS>
CLB_DEV Found search(Row &r, const Limit &among, u64 want, double share, bool allow_few, const float *largest = nullptr) {
  constexpr int SW = ST / 32, MOST = ST < CAP ? ST : CAP;
  Shared *sh = r.sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t lo = 0, hi = 0, shift = 0;   // the run that a level divides: at level 0 everything, then the keys [lo, hi]
  Found f{};
  bool quick = !MASS && largest;
  for (int level = 0;; ++level) {
    const bool whole = level == 0 && among.all();
    auto inside = [&](float x, uint32_t i) {
      if (whole) return true;
      const uint32_t k = key_of(x);
      return among.keeps(k, r.base + i) && (level == 0 || (k >= lo && k <= hi));
    };
    auto place = [&](float x) { return level == 0 ? r.bin(x) : (hi - key_of(x)) >> shift; };
    for (int b = tid; b < NB; b += ST) { sh->lo[b] = 0; sh->hi[b] = 0; }
    if (tid == 0) { sh->n_list = 0; sh->n_above = 0; }
    __syncthreads();
    if (MASS) {
      auto weigh = [&](uint32_t i, bool end) {
        float x[E];
        double w[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {   // what does not belong here weighs nothing
          const uint32_t q = i + e * ST;
          x[e] = !end || q < r.n ? r.x[q] : -INFINITY;
          if (!whole && !inside(x[e], q)) x[e] = -INFINITY;
        }
        r.weights(x, w);
#pragma unroll
        for (int e = 0; e < E; ++e) {   // in 32-bit halves with the carry, since only those add in one instruction
          if (!(x[e] > r.floor)) continue;
          const u64 m = units(w[e]);
          const uint32_t b = place(x[e]), l = static_cast<uint32_t>(m);
          const uint32_t up = static_cast<uint32_t>(m >> 32) + (atomicAdd(&sh->lo[b], l) > ~l ? 1u : 0u);
          if (up) atomicAdd(&sh->hi[b], up);
        }
      };
      uint32_t i = tid;
      for (; i + (E - 1) * ST < r.n; i += E * ST) weigh(i, false);
      if (i < r.n) weigh(i, true);
    } else if (quick) {
      atomicAdd(&sh->lo[r.bin(*largest)], 1u);
    } else {
#pragma unroll 4
      for (uint32_t i = tid; i < r.n; i += ST) {
        const float x = r.x[i];
        if (inside(x, i)) atomicAdd(&sh->lo[place(x)], 1u);
      }
    }
    __syncthreads();
    for (int c = warp; c < 32; c += SW) {   // a warp adds NB / 32 bins
      u64 v = 0;
#pragma unroll
      for (int b = 0; b < NB / 32; b += 32) v += (static_cast<u64>(sh->hi[NB / 32 * c + b + lane]) << 32) + sh->lo[NB / 32 * c + b + lane];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
      if (lane == 0) sh->coarse[c] = v;
    }
    cluster_sync<CL>();
    if (warp == 0) {   // the NB / 32 bins that hold the border, then the one, then its keys
      u64 v = 0;
#pragma unroll
      for (uint32_t c = 0; c < CL; ++c) v += remote<CL>(&sh->coarse[lane], c);
      u64 s = warp_scan(v);
      if (level == 0) {
        f.total = __shfl_sync(FULL_MASK, s, 31);
        if (MASS) {
          const double w = ceil(share * static_cast<double>(f.total));
          want = w >= static_cast<double>(f.total) ? f.total : w < 1.0 ? 1ull : static_cast<u64>(w);
        }
      }
      const int cb = min(__ffs(__ballot_sync(FULL_MASK, s >= want)) - 1, 31) & 31;
      const u64 before = __shfl_sync(FULL_MASK, s - v, cb);
      constexpr int PER = NB / 32 / 32;   // a lane's bins
      u64 bv[PER], mine = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int at = NB / 32 * cb + PER * lane + e;
        bv[e] = 0;
#pragma unroll
        for (uint32_t c = 0; c < CL; ++c) {
          bv[e] += remote<CL>(&sh->lo[at], c);
          if (MASS) bv[e] += static_cast<u64>(remote<CL>(&sh->hi[at], c)) << 32;
        }
        mine += bv[e];
      }
      s = before + warp_scan(mine);
      const int fl = min(__ffs(__ballot_sync(FULL_MASK, s >= want)) - 1, 31) & 31;
      u64 at = s - mine, value = bv[0];
      uint32_t b = NB / 32 * cb + PER * lane;
#pragma unroll
      for (int e = 1; e < PER; ++e)
        if (at + value < want) { at += value; value = bv[e]; ++b; }
      b = __shfl_sync(FULL_MASK, b, fl);   // the border's lane speaks for the warp: what follows is the warp's together
      at = __shfl_sync(FULL_MASK, at, fl);
      value = __shfl_sync(FULL_MASK, value, fl);
      // the bin's keys: bins do not grow with the key, so its ends are found by halving, 32 ways at a time
      uint32_t first, after;
      const uint32_t top_key = key_of(r.top);
      if (quick) {   // any prefix of the order that reaches past bin b will do: down to a logit just below the bin's
        first = key_of(cleaned(__fsub_rd(r.top, static_cast<float>(b + 1) * (1.0001f / BINS_PER_NAT) * r.heat)));
        after = top_key + 1;
      } else if (level == 0) {
        // the smallest key whose bin is at most b, and the smallest of the bins before it
        const bool to_top = b == 0 || (!MASS && allow_few && at + value <= MOST);   // all from `first` on are listed
        first = after = 0;
#pragma unroll 1
        for (int sh5 = 27; sh5 > -5; sh5 -= 5) {   // 5 bits a round, the last of 2
          const int sft = max(sh5, 0), ways = sh5 < 0 ? 4 : 32;
          auto reach = [&](uint32_t base, uint32_t most) {
            const uint32_t probe = base + ((static_cast<uint32_t>(lane) + 1) << sft) - 1;   // the last key of the lane's part
            return lane < ways && (probe >= top_key || (probe >= KEY_LOWEST && r.bin(logit_of(probe)) <= most));
          };
          const unsigned h0 = __ballot_sync(FULL_MASK, reach(first, b)), h1 = __ballot_sync(FULL_MASK, to_top || reach(after, b - 1));
          first += static_cast<uint32_t>(__ffs(h0) - 1) << sft;
          after += static_cast<uint32_t>(__ffs(h1) - 1) << sft;
        }
        if (b >= NB - 1) first = KEY_LOWEST;
        if (to_top) after = top_key + 1;
      } else {
        after = hi - (b << shift) + 1;
        first = after - (1u << shift) < lo || after < (1u << shift) ? lo : after - (1u << shift);
      }
      if (lane == fl) {
        sh->found[0] = (static_cast<u64>(after) << 32) | first;
        sh->found[1] = at;   // before the bin
        sh->found[2] = value;
        sh->found[3] = want;
        sh->found[4] = f.total;
      }
    }
    __syncthreads();
    const uint32_t k0 = static_cast<uint32_t>(sh->found[0]), k1 = static_cast<uint32_t>(sh->found[0] >> 32) - 1;   // the bin's keys: k0 .. k1
    const u64 before = sh->found[1];
    if (!quick) want = sh->found[3] - before;
    if (level == 0) f.total = sh->found[4];
    // list the bin's tokens and, where counts say that it fits, those before it
    const bool with_above = quick || (!MASS && allow_few && level == 0 && before + sh->found[2] <= MOST);
    const float x0 = logit_of(max(k0, KEY_LOWEST)), x1 = logit_of(k1 == 0x7fffffffu ? k1 - 1 : k1);   // (no -0)
    const bool every = among.all();
    auto list = [&](bool bin, bool above) {
      uint32_t seen = 0;
      auto look = [&](float x, uint32_t i) {   // (floats stand in the order of their keys)
        if (x < x0) return;
        const uint32_t k = key_of(x);
        if (!every && !among.keeps(k, r.base + i)) return;
        if (x <= x1 ? bin : above) {
          const uint32_t q = atomicAdd(&sh->n_list, 1u);
          if (q < MOST) sh->list[q] = token_word(k, r.base + i);
        } else {
          ++seen;
        }
      };
      uint32_t i = tid;
      for (; i + 3 * ST < r.n; i += 4 * ST) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = r.x[i + e * ST];
        if (fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) < x0) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) look(x[e], i + e * ST);
      }
      for (; i < r.n; i += ST) look(r.x[i], i);
      if (MASS && !above) {   // how many come before the bin
        seen = __reduce_add_sync(FULL_MASK, seen);
        if (lane == 0 && seen) atomicAdd(&sh->n_above, seen);
      }
    };
    list(true, with_above);
    cluster_sync<CL>();
    uint32_t n_bin = 0, n_above = 0;
#pragma unroll
    for (uint32_t c = 0; c < CL; ++c) {
      n_bin += remote<CL>(&sh->n_list, c);
      if (MASS) n_above += remote<CL>(&sh->n_above, c);
    }
    if (n_bin <= MOST) {
      f.few = with_above;
      if (MASS && allow_few && level == 0 && n_bin + n_above <= MOST) {
        cluster_sync<CL>();   // the counts have been read
        list(false, true);
        cluster_sync<CL>();
        f.few = true;
      }
      u64 x = gather<CL>(r, f.n);
      cluster_sync<CL>();   // lists and histograms have been read
      x = sort_words<MOST>(sh, x, static_cast<int>(f.n));
      f.word = x;
      if (f.few) return f;
      const uint32_t k = static_cast<uint32_t>(x >> 32);
      const u64 val = static_cast<uint32_t>(tid) < f.n ? (MASS ? r.mass(k) : 1ull) : 0ull;
      u64 t;
      const u64 s = block_scan<ST>(sh, val, t);
      if (s < want && s + val >= want) sh->found[5] = x;
      __syncthreads();
      const u64 w = sh->found[5];
      f.lim = Limit{static_cast<uint32_t>(w >> 32), 0xffffffffu - static_cast<uint32_t>(w)};
      return f;
    }
    if (quick) {   // too many: start over with all of them
      quick = false;
      level = -1;
      cluster_sync<CL>();   // lists and histograms have been read
      continue;
    }
    // the range of that bin's keys over the cluster
    uint32_t kmin = 0xffffffffu, kmax = 0;
    for (uint32_t i = tid; i < r.n; i += ST) {
      const uint32_t k = key_of(r.x[i]);
      if (k >= k0 && k <= k1 && among.keeps(k, r.base + i)) { kmin = min(kmin, k); kmax = max(kmax, k); }
    }
    kmin = __reduce_min_sync(FULL_MASK, kmin);
    kmax = __reduce_max_sync(FULL_MASK, kmax);
    __syncthreads();
    if (lane == 0) sh->part[warp] = (static_cast<u64>(kmax) << 32) | kmin;
    __syncthreads();
    if (warp == 0) {
      kmin = __reduce_min_sync(FULL_MASK, static_cast<uint32_t>(sh->part[lane % SW]));
      kmax = __reduce_max_sync(FULL_MASK, static_cast<uint32_t>(sh->part[lane % SW] >> 32));
      if (lane == 0) sh->mine[1] = (static_cast<u64>(kmax) << 32) | kmin;
    }
    cluster_sync<CL>();
    lo = 0xffffffffu;
    hi = 0;
#pragma unroll
    for (uint32_t c = 0; c < CL; ++c) {
      const u64 m = remote<CL>(&sh->mine[1], c);
      lo = min(lo, static_cast<uint32_t>(m));
      hi = max(hi, static_cast<uint32_t>(m >> 32));
    }
    if (lo == hi) {   // one key: the q-th of its tokens by id
      const u64 one = MASS ? r.mass(lo) : 1ull, q = one ? (want + one - 1) / one : 1;
      u64 c = 0, t, cl_total;
      const uint32_t i0 = min(tid * r.per_thread, r.n), i1 = min(i0 + r.per_thread, r.n);
      for (uint32_t i = i0; i < i1; ++i) c += key_of(r.x[i]) == lo && among.keeps(lo, r.base + i);
      u64 s = block_scan<ST>(sh, c, t);
      s += cluster_scan<CL>(r, t, cl_total);
      if (tid == 0) sh->mine[2] = 0;
      __syncthreads();
      if (s < q && s + c >= q)
        for (uint32_t i = i0; i < i1; ++i)
          if (key_of(r.x[i]) == lo && among.keeps(lo, r.base + i) && ++s == q) sh->mine[2] = r.base + i + 1ull;
      cluster_sync<CL>();
      u64 id = 0;
#pragma unroll
      for (uint32_t d = 0; d < CL; ++d) id = max(id, remote<CL>(&sh->mine[2], d));
      cluster_sync<CL>();
      f.few = false;
      f.lim = Limit{lo, static_cast<uint32_t>(id - 1)};
      return f;
    }
    const int bits = 32 - __clz(hi - lo);
    shift = bits > 11 ? bits - 11 : 0;   // NB = 2^11 bins
    cluster_sync<CL>();   // the ranges, lists and histograms have been read
  }
}

// n logits from src into shared memory, which starts where the first 16-byte boundary of src falls on one there too; returns the
// first's place. best: the thread's largest.
template <int ST, typename T>
CLB_DEV float *load_logits(const T *src, float *dst, uint32_t n, float &best) {
  constexpr uint32_t V = 16 / sizeof(T);
  auto clean = [&](float v) {
    v = cleaned(v);
    best = fmaxf(best, v);
    return v;
  };
  const uint32_t head = min(n, static_cast<uint32_t>(((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / sizeof(T)));
  dst += (4 - (head & 3)) & 3;
  if (threadIdx.x < head) dst[threadIdx.x] = clean(to_f32(src[threadIdx.x]));
  const uint32_t body = (n - head) / V;
  const uint4 *v = reinterpret_cast<const uint4 *>(src + head);
#pragma unroll 8
  for (uint32_t i = threadIdx.x; i < body; i += ST) {
    const uint4 w = __ldcs(v + i);
    const T *t = reinterpret_cast<const T *>(&w);
#pragma unroll
    for (uint32_t e = 0; e < V; e += 4)
      *reinterpret_cast<float4 *>(dst + head + V * i + e) = make_float4(clean(to_f32(t[e])), clean(to_f32(t[e + 1])), clean(to_f32(t[e + 2])), clean(to_f32(t[e + 3])));
  }
  const uint32_t rest = head + V * body + threadIdx.x;
  if (rest < n) dst[rest] = clean(to_f32(src[rest]));
  return dst;
}

// One row by CL CTAs: its logits lie in their shared memory, a slice each, and are read from memory once.
template <int CL, int ST>
__global__ void __launch_bounds__(ST, CL == 1 ? 1024 / ST : 1) sample_kernel(const clb200_sampling s, const uint32_t slice) {
  constexpr int SW = ST / 32, MOST = ST < CAP ? ST : CAP;
  extern __shared__ __align__(16) uint8_t sm[];
  Shared *sh = reinterpret_cast<Shared *>(sm);
  float *room = reinterpret_cast<float *>(sh + 1);   // slice + 3
  const int row = blockIdx.x / CL, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Row r;
  r.sh = sh;
  r.rank = cluster_rank<CL>();
  r.base = r.rank * slice;
  r.n = r.base < static_cast<uint32_t>(s.vocab) ? min(slice, static_cast<uint32_t>(s.vocab) - r.base) : 0;
  r.per_thread = ((slice + ST - 1) / ST) | 1;   // odd: a warp's threads read different banks
  const float t = s.temperature ? s.temperature[row] : 1.f, share = s.top_p ? s.top_p[row] : 1.f, least = s.min_p ? s.min_p[row] : 0.f, draw = s.u[row];
  const int k = s.top_k ? s.top_k[row] : 0;
  if (tid < 128) sh->exp2_128[tid] = __hiloint2double(__double2hiint(EXP2_128[tid]) - (tid << 13), __double2loint(EXP2_128[tid]));
  float best = -INFINITY;
  const int64_t at = row * s.stride + r.base;
  if (s.type == T_F32) r.x = load_logits<ST>(static_cast<const float *>(s.logits) + at, room, r.n, best);
  else if (s.type == T_F16) r.x = load_logits<ST>(static_cast<const __half *>(s.logits) + at, room, r.n, best);
  else r.x = load_logits<ST>(static_cast<const __nv_bfloat16 *>(s.logits) + at, room, r.n, best);
  auto largest = [&](u64 v, bool again) {   // of the row's threads
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(FULL_MASK, v, o));
    __syncthreads();
    if (lane == 0) sh->part[tid >> 5] = v;
    __syncthreads();
    v = sh->part[lane % SW];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(FULL_MASK, v, o));
    if constexpr (CL > 1) {
      if (again) cluster_sync<CL>();   // what was exchanged before has been read
      if (tid == 0) sh->mine[3] = v;
      cluster_sync<CL>();
#pragma unroll
      for (uint32_t c = 0; c < CL; ++c) v = max(v, remote<CL>(&sh->mine[3], c));
    }
    return v;
  };
  r.top = logit_of(static_cast<uint32_t>(largest(key_of(best), false)));
  if (r.top == -INFINITY || !(t > 0.f)) {
    u64 first = 0;   // the lowest id among the largest
    for (uint32_t i = tid; i < r.n; i += ST)
      if (r.x[i] == r.top) { first = 0xffffffffu - (r.base + i); break; }
    first = largest(first, true);
    if (r.rank == 0 && tid == 0) {
      s.token[row] = r.top == -INFINITY ? -1 : static_cast<int>(0xffffffffu - static_cast<uint32_t>(first));
      if (s.prob) s.prob[row] = r.top == -INFINITY ? 0.f : 1.f;
    }
    cluster_sync<CL>();   // the others may still be reading this CTA's shared memory
    return;
  }
  if (r.top == INFINITY) {   // those at infinity share everything
    for (uint32_t i = tid; i < r.n; i += ST) r.x[i] = r.x[i] == INFINITY ? 0.f : -INFINITY;
    r.top = 0.f;
    best = best == INFINITY ? 0.f : -INFINITY;
    __syncthreads();
  }
  r.half_top = 0.5f * r.top;
  r.top_d = static_cast<double>(r.top);
  const float heat = r.heat = fmaxf(t, 1.17549435e-38f);   // the smallest normal number, whose inverse is finite
  r.inv_f = 1.0f / heat;
  r.scale = 1.4426950408889634 / static_cast<double>(heat);
  // 64 temperatures below the largest, where a weight is below 2^-92; where rounding comes in (steps of h >= 128 temperatures / 3)
  // still at least 42 temperatures, below 2^-60.
  r.floor = fminf(fmaf(-64.f, heat, r.top), nextafterf(r.top, -INFINITY));
  const double min_w = least > 0.f ? fmin(static_cast<double>(least), 1.0) : 0.0;
  const double u = fmin(fmax(static_cast<double>(draw), 0.0), 1.0);   // a NaN counts as 0
  const bool by_k = k > 0 && k < s.vocab, by_p = share < 1.f;
  auto border = [](double part, u64 total) { return min(static_cast<u64>(part * static_cast<double>(total)), total - 1); };
  auto answer = [&](uint32_t id, double w, u64 total) {
    s.token[row] = static_cast<int>(id);
    if (s.prob) s.prob[row] = static_cast<float>(w / (static_cast<double>(total) * (1.0 / UNIT)));
  };
  Limit lim{KEY_LOWEST, 0xffffffffu};
  if (by_k || by_p) {
    // each thread has several tokens and their largest ones are more than enough
    const float *quick = by_k && k <= MOST / 2 && s.vocab >= 4 * CL * ST ? &best : nullptr;
    Found f = by_k ? search<CL, ST, false>(r, lim, static_cast<u64>(k), 0.0, true, quick) : search<CL, ST, true>(r, lim, 0, static_cast<double>(share), true);
    if (f.few) {   // the candidates, sorted, a thread each: the filters are prefixes, the draw goes by id
      const uint32_t q = static_cast<uint32_t>(f.word >> 32), id = 0xffffffffu - static_cast<uint32_t>(f.word);
      const bool cand = static_cast<uint32_t>(tid) < f.n && (!by_k || tid < k);
      double w = cand ? r.weight(logit_of(q)) : 0.0;
      u64 m = units(w), total, kept;
      const u64 before = block_scan<ST>(sh, m, total);
      if (by_p) {
        if (!by_k) total = f.total;
        const double x = ceil(static_cast<double>(share) * static_cast<double>(total));
        const u64 want = x >= static_cast<double>(total) ? total : x < 1.0 ? 1ull : static_cast<u64>(x);
        if (before >= want) m = 0;
      }
      if (w < min_w) m = 0;
      __syncthreads();
      if (tid < MOST) sh->list[tid] = m;
      __syncthreads();
      // by id: the complement of the id above, the place below
      const u64 x = sort_words<MOST>(sh, m ? (static_cast<u64>(0xffffffffu - id) << 32) | static_cast<uint32_t>(tid) : 0ull, by_k ? min(static_cast<int>(f.n), k) : static_cast<int>(f.n));
      const uint32_t place = static_cast<uint32_t>(x);
      m = x ? sh->list[place & (MOST - 1)] : 0;
      const u64 s0 = block_scan<ST>(sh, m, kept);
      const u64 want = border(u, kept);
      if (r.rank == 0 && s0 <= want && want < s0 + m) {
        const uint32_t token = 0xffffffffu - static_cast<uint32_t>(x >> 32);
        sh->found[0] = token;
        sh->found[1] = place;
        sh->found[2] = kept;
      }
      __syncthreads();
      if (r.rank == 0 && tid == static_cast<int>(sh->found[1])) answer(static_cast<uint32_t>(sh->found[0]), w, sh->found[2]);
      cluster_sync<CL>();
      return;
    }
    lim = f.lim;
    if (by_k && by_p) lim = search<CL, ST, true>(r, lim, 0, static_cast<double>(share), false).lim;
  }
  // The kept masses by id: a warp takes a run of the slice, 32 E tokens at a time. The sums of the warps and CTAs before it say
  // which warp goes through its run once more.
  constexpr uint32_t STEP = 32 * E;
  const float lowest = logit_of(lim.key);
  const uint32_t run = (slice + SW * STEP - 1) / (SW * STEP) * STEP, i0 = min(warp * run, r.n), i1 = min(i0 + run, r.n);
  float x[E];
  double w[E];
  auto weigh = [&](uint32_t i) {   // the sum of the lane's
    bool any = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t q = i + 32 * e + lane;
      x[e] = q < i1 ? r.x[q] : -INFINITY;
      if (x[e] < lowest || (x[e] == lowest && r.base + q > lim.id)) x[e] = -INFINITY;
      any = any || x[e] != -INFINITY;
    }
    u64 sum = 0;
    if (!__any_sync(FULL_MASK, any)) return sum;
    r.weights(x, w);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      w[e] = w[e] >= min_w ? w[e] : 0.0;
      sum += units(w[e]);
    }
    return sum;
  };
  u64 mine = 0, cta_total, total;
  for (uint32_t i = i0; i < i1; i += STEP) mine += weigh(i);
  u64 before = block_scan<ST>(sh, mine, cta_total);
  const u64 after = cluster_scan<CL>(r, cta_total, total) + __shfl_sync(FULL_MASK, before + mine, 31);
  before += after - __shfl_sync(FULL_MASK, before + mine, 31);
  before = __shfl_sync(FULL_MASK, before, 0);
  const u64 want = border(u, total);
  if (before <= want && want < after) {
    for (uint32_t i = i0; i < i1; i += STEP) {
      u64 sum = weigh(i);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL_MASK, sum, o);
      if (before + sum <= want) {
        before += sum;
        continue;
      }
      bool done = false;
#pragma unroll
      for (int e = 0; e < E; ++e) {   // (a step that is reached has weights)
        const u64 m = units(w[e]), v = before + warp_scan(m);
        if (!done && v - m <= want && want < v) answer(r.base + i + 32 * e + lane, w[e], total);
        before = __shfl_sync(FULL_MASK, v, 31);
        done = done || want < before;
      }
      break;
    }
  }
  cluster_sync<CL>();
}

template <int CL, int ST>
cudaError_t launch_sample(const clb200_sampling &s, int device, cudaStream_t st) {
  const uint32_t slice = (static_cast<uint32_t>(s.vocab) + CL - 1) / CL;
  static bool done[64] = {};
  if (device >= 64 || !done[device]) {
    const cudaError_t e = cudaFuncSetAttribute(sample_kernel<CL, ST>, cudaFuncAttributeMaxDynamicSharedMemorySize, SAMPLE_SMEM);
    if (e != cudaSuccess) return e;
    if (device < 64) done[device] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(s.rows) * CL);
  cfg.blockDim = dim3(ST);
  cfg.dynamicSmemBytes = sizeof(Shared) + static_cast<size_t>(slice + 3) * 4;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CL;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<CL, ST>, s, slice);
}

template <int ST>
cudaError_t launch_cl(int cl, const clb200_sampling &s, int device, cudaStream_t st) {
  switch (cl) {
    case 1: return launch_sample<1, ST>(s, device, st);
    case 2: return launch_sample<2, ST>(s, device, st);
    case 4: return launch_sample<4, ST>(s, device, st);
    default: return launch_sample<8, ST>(s, device, st);
  }
}

int check(const clb200_sampling *s, char *err, size_t errlen) {
  if (!s) { errf(err, errlen, "no arguments"); return 1; }
  if (s->rows < 0 || s->rows > (1 << 24) || s->vocab < 1 || s->vocab > SAMPLE_MAX_VOCAB) {
    errf(err, errlen, "%d rows of %d logits: takes 1 to %d logits a row", s->rows, s->vocab, SAMPLE_MAX_VOCAB);
    return 1;
  }
  if (s->type != T_F32 && s->type != T_F16 && s->type != T_BF16) { errf(err, errlen, "logits are %s: F32, F16 or BF16", type_name(s->type)); return 1; }
  if (s->rows > 0 && (!s->logits || !s->u || !s->token)) { errf(err, errlen, "a buffer is missing"); return 1; }
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
  // The fewest CTAs that hold a row, since the exchange costs more than it saves once the SMs are busy (256 rows of 50304: 89 us
  // with one a row, 123 with two, 190 with four), and more of them for long rows while that leaves no row waiting (a GPC takes two
  // clusters of eight: 17 rows of 151936 take 23 us with four each and 33 with eight; filters want few CTAs, sums over everything
  // many: 8 rows of 14678 with top-k 17.4 us with one, 20.0 with four; 15 rows of 39554 without filters 15.6 with one, 11.2 with
  // four). Threads: barriers and scans cost less with fewer, passes over the logits less with more (one row of 151936 by eight CTAs:
  // 15.0 us with 512 threads, 19.4 with 1024, 16 with 256; 100 rows of 32000: 39 and 34 with 1024), and small CTAs share an SM (1000
  // rows of 10000: 47 us with 256, 57 with 512, 91 with 1024; 140 rows of 6000, which need not: 18.2, 16.3, 17.9).
  cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : c->stream;
  int cl = 1;
  while (cl < 8 && ((s->vocab + cl - 1) / cl > static_cast<int>(MAX_SLICE) || (static_cast<int64_t>(s->rows) * cl * 2 <= 128 && s->vocab >= 12288 * cl))) cl *= 2;
  cudaError_t e;
  if (s->vocab <= 2560 || (s->vocab <= 10240 && s->rows > c->sms)) e = launch_sample<1, 256>(*s, c->device, st);
  else if (s->vocab <= 20480 * cl) e = launch_cl<512>(cl, *s, c->device, st);
  else e = launch_cl<1024>(cl, *s, c->device, st);
  CUDA_OR(e, "launching the sampling");
  return 0;
}
