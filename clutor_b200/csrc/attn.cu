// clb200_attention: attention of chunks of new tokens over a paged key/value cache. This file holds the entry point, the kernel
// for few rows per key/value head and the one that joins partial results; attn.cuh how work is divided, attn_tc.cu the kernel for
// many rows.
//
// out = sum_j p_j v_j with p the softmax of the scaled scores of the visible positions, in one pass over the keys and values: a
// row keeps the maximum m of its scores so far (in units of 1 / log2 e), the sum l of 2^(x - m) and the unnormalised values, and
// scales l and the values by 2^(m - m') when a tile raises m to m'. Partial results of one row, (m, l, values) of disjoint sets of
// positions, join by the same rule.
#include <algorithm>

#include "attn.cuh"
#include "ctx.cuh"
#include "serve.cuh"

namespace clb {
namespace {

// ---- few rows: mma.sync ----------------------------------------------------------------------------------------------------

// Up to 16 x MT rows (new tokens x query heads of a key/value head): bound by the bytes of the cache, each read once. A warp
// takes 16 positions of every tile of 64 through a ring of its own (cp.async, so positions past the sequence's end come as zeros
// whatever the slots hold) and keeps its own (m, l, values) for them, so warps do not wait on one another inside an item; their
// states are joined at its end, under the first loads of the next item (200 sequences of up to 300 positions, 32 heads over 8:
// 40 us, 45 with those loads behind the join; the states handed from warp to warp through one buffer instead: 50). Products on
// m16n8k16: at 8 of 16 rows in use they are far from the limit, while eight warps an SM with two stages each on their way cover
// HBM's latency. 64 sequences of up to 8000 positions, 32 heads over 4 of 128: 104 us = 6.06 TB/s, 92 % of the measured copy
// rate; one token over 500 positions 8.9 us with the join.
constexpr int RT = 128, RW = RT / 32, RN = 16 * RW;   // threads, warps, positions per tile (16 per warp)

template <int HD, int MT>
struct RowsShape {
  static constexpr int ROWS = 16 * MT;
  static constexpr int STAGES = HD == 64 ? 6 : 3;
  static constexpr uint32_t HALF = 16 * HD * 2, STAGE = 2 * HALF;         // a warp's keys (then values) of one tile
  static constexpr uint32_t Q = ROWS * HD * 2, KV = RW * STAGES * STAGE;
  static constexpr uint32_t SMEM = Q + KV + RW * 16 * 8;
  static constexpr int PER_SM = HD == 256 ? 1 : 2;
  static_assert(16 * HD * 4 <= STAGE, "a warp's values of 16 rows fit a stage");
  static_assert((ATTN_MAX_SEQ + 1) * 8 <= static_cast<int>(KV), "the prefix sums fit the stages");
};

CLB_DEV void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
CLB_DEV void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename C>
CLB_DEV void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(C) == 2 && __is_same(C, __half))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte offset of 16-byte chunk c of row r in rows of HD half-precision elements; eight rows' equal chunks in eight bank groups.
template <int HD>
CLB_DEV uint32_t chunk_at(int r, int c) { return static_cast<uint32_t>(r * HD * 2 + ((c ^ (r & 7)) << 4)); }

template <typename C, typename O, int HD, int MT>
__global__ void __launch_bounds__(RT, RowsShape<HD, MT>::PER_SM) attn_rows_kernel(const AttnArgs g) {
  using S = RowsShape<HD, MT>;
  constexpr int KK = HD / 16, ROWS = S::ROWS;
  constexpr bool QREG = MT * KK <= 8;   // the query fragments stay in registers
  extern __shared__ __align__(128) uint8_t sm[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
  const clb200_attn &a = g.a;
  const clb200_kv &kv = g.kv;
  const uint32_t q_sm = smem_addr(sm), kv_sm = q_sm + S::Q + warp * S::STAGES * S::STAGE;
  float2 *states = reinterpret_cast<float2 *>(sm + S::Q + S::KV);   // [RW][16] a warp's maximum and sum of a row
  const float sc = a.scale * LOG2E;
  const int gr = lane >> 2, gc = (lane & 3) * 2;   // the lane's row and first column in an accumulator
  if (tid == 0) g.joins[cta] = make_int4(0, 0, 0, 0);
  int64_t *prefix = reinterpret_cast<int64_t *>(sm + S::Q);
  attn_prefix<RN>(g, prefix, cta);
  AttnRun<RN> run;
  run.init(g, prefix, cta);
  __syncthreads();   // the prefix sums have been read: the stages take their place
  AttnSpan span;
  int n = 0, i0 = 0, base = 0;   // the item's tiles, its first, and the stage of that one
  auto issue = [&](int i) {   // this warp's 16 positions of tile i of the item
    if (i < n) {
      const int j0 = span.tile(i0 + i) * RN + warp * 16;
      if (j0 <= span.hi) {
        const AttnSlot at0 = attn_hidden(g, span.lo, j0, 16) ? AttnSlot{-1, 0} : attn_slot(g, run.s, j0);
        const int64_t from = (at0.page < 0 ? 0 : at0.page * kv.page_stride + at0.slot * kv.slot_stride) + run.head * kv.head_stride;
        const uint32_t dst = kv_sm + (base + i) % S::STAGES * S::STAGE;
        const int left = at0.page < 0 ? 0 : run.q.kv - j0;   // positions behind the sequence's end come as zeros
#pragma unroll
        for (int e = lane; e < 16 * (HD / 8); e += 32) {
          const int r = e / (HD / 8), c = e % (HD / 8);
          const int64_t at = r < left ? from + r * kv.slot_stride + 8 * c : 0;
          cp_async16(dst + chunk_at<HD>(r, c), static_cast<const C *>(kv.k) + at, r < left);
          cp_async16(dst + S::HALF + chunk_at<HD>(r, c), static_cast<const C *>(kv.v) + at, r < left);
        }
      }
    }
    cp_commit();
  };
  // The next item with tiles for this CTA becomes the current one; its queries and first tiles are sent for.
  auto begin = [&]() {   // false at the end of the run
    for (n = 0; run.more(); run.advance(g, span)) {
      span = attn_span<RN>(g, run.q, run.qt);
      i0 = run.first(g);
      n = run.tiles(g, span);
      if (n) break;   // else the run ends in the item's lead
    }
    if (n == 0) return false;
    const int t0 = run.qt * g.tpi;
    for (int i = tid; i < ROWS * (HD / 8); i += RT) {
      const int r = i / (HD / 8), c = i % (HD / 8), tr = attn_token(g, r), t = t0 + tr, h = run.head * g.group + r - tr * g.group;
      const bool live = r < g.tpi * g.group && t < run.q.nq;
      cp_async16(q_sm + chunk_at<HD>(r, c), static_cast<const C *>(a.q) + (live ? (run.q.row + t) * a.q_stride + h * HD + 8 * c : 0), live);
    }
    cp_commit();
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; ++i) issue(i);
    return true;
  };
  bool more = begin();
  while (more) {
    cp_wait<S::STAGES - 1>();   // the queries
    __syncthreads();
    uint32_t qf[QREG ? MT : 1][QREG ? KK : 1][4];
    auto load_q = [&](int mt, int kk, uint32_t (&f)[4]) {
      ldsm4(f, q_sm + chunk_at<HD>(16 * mt + (lane & 15), 2 * kk + (lane >> 4)));
    };
    if constexpr (QREG)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) load_q(mt, kk, qf[mt][kk]);
    float o[MT][HD / 8][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt][0] = m[mt][1] = -INFINITY;
      l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
      for (int d = 0; d < HD / 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][d][e] = 0.f;
    }
    for (int i = 0; i < n; ++i) {
      cp_wait<S::STAGES - 2>();
      __syncwarp();
      const int j0 = span.tile(i0 + i) * RN + warp * 16;
      if (j0 <= span.hi) {
        const uint32_t ks = kv_sm + (base + i) % S::STAGES * S::STAGE, vs = ks + S::HALF;
        float x[MT][2][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[mt][e >> 2][e & 3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          uint32_t b[4];
          ldsm4(b, ks + chunk_at<HD>((lane >> 4) * 8 + (lane & 7), 2 * kk + ((lane >> 3) & 1)));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            if constexpr (QREG) {
              mma16816<C>(x[mt][0], qf[mt][kk], b[0], b[1]);
              mma16816<C>(x[mt][1], qf[mt][kk], b[2], b[3]);
            } else {
              uint32_t f[4];
              load_q(mt, kk, f);
              mma16816<C>(x[mt][0], f, b[0], b[1]);
              mma16816<C>(x[mt][1], f, b[2], b[3]);
            }
          }
        }
        // some row does not see all 16 positions
        const bool edge = j0 + 15 > span.lo || (a.window > 0 && j0 <= span.hi - a.window && j0 + 15 >= a.sinks);
        uint32_t p[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[mt][e >> 2][e & 3] *= sc;
          if (edge) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int r = 16 * mt + gr + ((e & 2) ? 8 : 0), j = j0 + (e >> 2) * 8 + gc + (e & 1);
              if (!attn_sees(g, span.lo + attn_token(g, r), j)) x[mt][e >> 2][e & 3] = -INFINITY;
            }
          }
          float mx[2] = {m[mt][0], m[mt][1]};
#pragma unroll
          for (int e = 0; e < 8; ++e) mx[(e >> 1) & 1] = fmaxf(mx[(e >> 1) & 1], x[mt][e >> 2][e & 3]);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            mx[w] = fmaxf(mx[w], __shfl_xor_sync(FULL_MASK, mx[w], 1));
            mx[w] = fmaxf(mx[w], __shfl_xor_sync(FULL_MASK, mx[w], 2));
          }
          if (__any_sync(FULL_MASK, mx[0] > m[mt][0] || mx[1] > m[mt][1])) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const float f = m[mt][w] == -INFINITY ? 0.f : exp2_approx(m[mt][w] - mx[w]);
              l[mt][w] *= f;
              m[mt][w] = mx[w];
#pragma unroll
              for (int d = 0; d < HD / 8; ++d) { o[mt][d][2 * w] *= f; o[mt][d][2 * w + 1] *= f; }
            }
          }
          const float z[2] = {m[mt][0] == -INFINITY ? 0.f : m[mt][0], m[mt][1] == -INFINITY ? 0.f : m[mt][1]};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float &v = x[mt][e >> 2][e & 3];
            v = exp2_approx(v - z[(e >> 1) & 1]);
            l[mt][(e >> 1) & 1] += v;
          }
          // the probabilities are rounded to the cache's type, the type of the matrix product's operands
          p[mt][0] = pack2<C>(x[mt][0][0], x[mt][0][1]);
          p[mt][1] = pack2<C>(x[mt][0][2], x[mt][0][3]);
          p[mt][2] = pack2<C>(x[mt][1][0], x[mt][1][1]);
          p[mt][3] = pack2<C>(x[mt][1][2], x[mt][1][3]);
        }
#pragma unroll
        for (int d = 0; d < KK; ++d) {
          uint32_t b[4];
          ldsm4t(b, vs + chunk_at<HD>((lane & 7) + ((lane >> 3) & 1) * 8, 2 * d + (lane >> 4)));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma16816<C>(o[mt][2 * d], p[mt], b[0], b[1]);
            mma16816<C>(o[mt][2 * d + 1], p[mt], b[2], b[3]);
          }
        }
      }
      __syncwarp();   // the stage has been read by every lane
      issue(i + S::STAGES - 1);
    }
    // what the join needs of this item, then the next one's first loads
    const int row = run.q.row + run.qt * g.tpi, tokens = min(g.tpi, run.q.nq - run.qt * g.tpi), head = run.head;
    const bool whole = n == span.nt;
    const int slot = 2 * cta + (i0 == 0 ? 1 : 0);
    if (!whole && i0 == 0 && tid == 0) g.joins[cta] = make_int4(row, tokens, head, run.pieces(span.nt - n));
    base = (base + n) % S::STAGES;
    run.advance(g, span);
    // The warps' states (maximum and sum of each row, values in fp32), 16 rows at a time, each in the stage that the warp's next
    // item takes last; then joined in warp order.
    const uint32_t spare = (base + S::STAGES - 1) % S::STAGES * S::STAGE;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float *mine = reinterpret_cast<float *>(sm + S::Q + warp * S::STAGES * S::STAGE + spare);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        l[mt][w] += __shfl_xor_sync(FULL_MASK, l[mt][w], 1);
        l[mt][w] += __shfl_xor_sync(FULL_MASK, l[mt][w], 2);
        if ((lane & 3) == 0) states[warp * 16 + gr + 8 * w] = make_float2(m[mt][w], l[mt][w]);
#pragma unroll
        for (int d = 0; d < HD / 8; ++d)   // four rows' pairs in four groups of banks
          *reinterpret_cast<float2 *>(mine + (gr + 8 * w) * HD + 8 * (d ^ (gr & 3)) + gc) = make_float2(o[mt][d][2 * w], o[mt][d][2 * w + 1]);
      }
      __syncthreads();   // (the queries, too, have been read)
      if (mt == 0) {
        more = begin();
        if (!more) grid_launch_dependents();
      }
      for (int i = tid; i < 16 * (HD / 4); i += RT) {
        const int rr = i / (HD / 4), c = 4 * (i % (HD / 4)), r = 16 * mt + rr, tr = attn_token(g, r);
        if (r >= g.tpi * g.group || tr >= tokens) continue;
        float mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < RW; ++w) mm = fmaxf(mm, states[w * 16 + rr].x);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < RW; ++w) {
          const float2 st = states[w * 16 + rr];
          const float f = st.x == -INFINITY ? 0.f : exp2_approx(st.x - mm);
          const float4 u = *reinterpret_cast<const float4 *>(sm + S::Q + w * S::STAGES * S::STAGE + spare + 4 * (rr * HD + (c ^ ((rr & 3) << 3))));
          ll = fmaf(f, st.y, ll);
          v.x = fmaf(f, u.x, v.x); v.y = fmaf(f, u.y, v.y); v.z = fmaf(f, u.z, v.z); v.w = fmaf(f, u.w, v.w);
        }
        if (whole) {
          store4<O>(static_cast<O *>(a.out) + (row + tr) * a.out_stride + (head * g.group + r - tr * g.group) * HD + c, v, ll > 0.f ? 1.0f / ll : 0.f);
        } else {
          *reinterpret_cast<float4 *>(g.piece_o + (static_cast<int64_t>(slot) * g.rows + r) * HD + c) = v;
          if (c == 0) g.piece_ml[static_cast<int64_t>(slot) * g.rows + r] = make_float2(mm, ll);
        }
      }
      if (mt + 1 < MT) __syncthreads();   // these have been read
    }
  }
  cp_wait<0>();
}

// ---- joining the pieces of items that fell into several runs ---------------------------------------------------------------

constexpr int JT = 256;

// HD / 4 threads hold a row, four elements each. BY_ROW: a CTA takes as many rows as it has such groups, each going through the
// pieces in run order (many rows in few pieces: the prompt kernel's). Else a CTA takes one row, its groups every so-many-th piece,
// and their states are joined in group order (few rows in many pieces: a long cache's; with 128 threads 1.4 us slower there and as
// much faster at 64 sequences). Most CTAs find nothing and end; as many as max_q allows are launched (one token over 500 positions
// 8.9 us, 9.4 with CTAs for every row that an item could have).
template <typename O, int HD, bool BY_ROW>
__global__ void __launch_bounds__(JT) attn_join_kernel(const AttnArgs g) {
  constexpr int TPR = HD / 4, GROUPS = JT / TPR;
  __shared__ float4 sum[BY_ROW ? 1 : GROUPS][TPR];
  __shared__ float2 state[GROUPS];
  const int grp = threadIdx.x / TPR, e = threadIdx.x % TPR;
  const int r = BY_ROW ? blockIdx.y * GROUPS + grp : blockIdx.y;
  grid_dependency_wait();
  const int4 j = g.joins[blockIdx.x];
  const int tr = attn_token(g, r);
  if (j.w == 0 || tr >= j.y) return;   // no item, or no such row (of the whole CTA, where its threads meet below)
  // piece i: slot 1 of this CTA, then slot 0 of the CTAs that follow
  auto slot = [&](int i) { return static_cast<int64_t>(i == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + i)) * g.rows + r; };
  float m = -INFINITY, l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int U = 4;   // pieces on their way at once
  for (int i0 = BY_ROW ? 0 : grp; i0 <= j.w; i0 += U * (BY_ROW ? 1 : GROUPS)) {
    float2 ml[U];
    float4 o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * (BY_ROW ? 1 : GROUPS);
      ml[u] = make_float2(-INFINITY, 0.f);
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i <= j.w) {
        ml[u] = g.piece_ml[slot(i)];
        o[u] = *reinterpret_cast<const float4 *>(g.piece_o + slot(i) * HD + 4 * e);
      }
    }
    float mm = m;
#pragma unroll
    for (int u = 0; u < U; ++u) mm = fmaxf(mm, ml[u].x);
    const float f0 = m == -INFINITY ? 0.f : exp2_approx(m - mm);
    l *= f0;
    v.x *= f0; v.y *= f0; v.z *= f0; v.w *= f0;
    m = mm;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float f = ml[u].x == -INFINITY ? 0.f : exp2_approx(ml[u].x - mm);
      l = fmaf(f, ml[u].y, l);
      v.x = fmaf(f, o[u].x, v.x); v.y = fmaf(f, o[u].y, v.y); v.z = fmaf(f, o[u].z, v.z); v.w = fmaf(f, o[u].w, v.w);
    }
  }
  if constexpr (!BY_ROW) {
    sum[grp][e] = v;
    if (e == 0) state[grp] = make_float2(m, l);
    __syncthreads();
    if (grp != 0) return;
    for (int k = 0; k < GROUPS; ++k) m = fmaxf(m, state[k].x);
    l = 0.f;
    v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < GROUPS; ++k) {
      const float f = state[k].x == -INFINITY ? 0.f : exp2_approx(state[k].x - m);
      const float4 o = sum[k][e];
      l = fmaf(f, state[k].y, l);
      v.x = fmaf(f, o.x, v.x); v.y = fmaf(f, o.y, v.y); v.z = fmaf(f, o.z, v.z); v.w = fmaf(f, o.w, v.w);
    }
  }
  store4<O>(static_cast<O *>(g.a.out) + (j.x + tr) * g.a.out_stride + (j.z * g.group + r - tr * g.group) * HD + 4 * e, v, l > 0.f ? 1.0f / l : 0.f);
}

// ---- host ------------------------------------------------------------------------------------------------------------------

template <typename C, typename O, int HD, int MT>
cudaError_t launch_rows(const AttnArgs &g, cudaStream_t st) {
  using S = RowsShape<HD, MT>;
  static bool done[64] = {};
  const cudaError_t e = allow_smem(attn_rows_kernel<C, O, HD, MT>, S::SMEM, done);
  if (e != cudaSuccess) return e;
  attn_rows_kernel<C, O, HD, MT><<<g.nc, RT, S::SMEM, st>>>(g);
  return cudaGetLastError();
}

template <typename O, int HD>
cudaError_t launch_join(const AttnArgs &g, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  const bool by_row = g.rows > 32;
  const int groups = JT / (HD / 4), rows = std::max(std::min(g.tpi, g.a.max_q), 1) * g.group;   // the most that an item can have
  cfg.gridDim = dim3(g.nc, by_row ? (rows + groups - 1) / groups : rows);
  cfg.blockDim = dim3(JT);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return by_row ? cudaLaunchKernelEx(&cfg, attn_join_kernel<O, HD, true>, g) : cudaLaunchKernelEx(&cfg, attn_join_kernel<O, HD, false>, g);
}

template <typename C, typename O, int HD>
cudaError_t launch_all(const AttnArgs &g, cudaStream_t st) {
  cudaError_t e;
  if (g.rows > 32) e = launch_attn_tc(g, st);
  else if (g.rows == 16) e = launch_rows<C, O, HD, 1>(g, st);
  else if constexpr (HD <= 128) e = launch_rows<C, O, HD, 2>(g, st);
  else e = cudaErrorInvalidValue;
  return e != cudaSuccess ? e : launch_join<O, HD>(g, st);
}

template <typename C, typename O>
cudaError_t launch_hd(const AttnArgs &g, cudaStream_t st) {
  switch (g.kv.head_dim) {
    case 64: return launch_all<C, O, 64>(g, st);
    case 128: return launch_all<C, O, 128>(g, st);
    default: return launch_all<C, O, 256>(g, st);
  }
}

// The kernel's shape for a call, and its workspace: partial values, their maxima and sums, the list of items to join.
struct AttnPlan {
  int rows, tpi, nc;
  size_t off_ml, off_joins, total;
};
AttnPlan attn_plan(int sms, const clb200_kv &kv, const clb200_attn &a) {
  AttnPlan p{};
  const int group = a.n_head / kv.n_kv;
  const int64_t need = a.max_q * static_cast<int64_t>(group);
  p.rows = need <= 16 ? 16 : need <= 32 && kv.head_dim <= 128 ? 32 : attn_tc_rows(kv.head_dim);
  p.nc = sms * (p.rows <= 32 && kv.head_dim <= 128 ? 2 : 1);
  p.tpi = p.rows <= 32 ? p.rows / group : p.rows / 128 * (128 / group);
  const size_t pieces = static_cast<size_t>(p.nc) * 2 * p.rows;
  p.off_ml = al(pieces * kv.head_dim * 4);
  p.off_joins = p.off_ml + al(pieces * 8);
  p.total = p.off_joins + al(static_cast<size_t>(p.nc) * 16);
  return p;
}

int check(const clb200_kv *kv, const clb200_attn *a, char *err, size_t errlen) {
  if (!kv || !a) { errf(err, errlen, "no cache or arguments"); return 1; }
  if (check_kv(kv, err, errlen)) return 1;
  if (a->T < 0 || a->n_head < 1 || a->n_head % kv->n_kv || a->n_head / kv->n_kv > ATTN_MAX_GROUP) {
    errf(err, errlen, "%d rows of %d query heads over %d key/value heads: the query heads must be a multiple of them, at most %d times as many",
         a->T, a->n_head, kv->n_kv, ATTN_MAX_GROUP);
    return 1;
  }
  if (a->max_q < 0) { errf(err, errlen, "max_q %d", a->max_q); return 1; }
  if (a->out_type != T_F32 && a->out_type != kv->type) { errf(err, errlen, "out is %s: it must be F32 or the cache's type", type_name(a->out_type)); return 1; }
  if (a->T > 0 && (!a->q || !a->out)) { errf(err, errlen, "a buffer is missing"); return 1; }
  if (!(a->scale > 0.f) || a->scale > 3.0e38f) { errf(err, errlen, "scale %g: a positive number", a->scale); return 1; }
  if (a->window < 0 || a->sinks < 0) { errf(err, errlen, "window %d, sinks %d: not negative", a->window, a->sinks); return 1; }
  const int64_t nq = static_cast<int64_t>(a->n_head) * kv->head_dim;
  if (a->q_stride < nq || a->out_stride < nq || a->q_stride % 8 || a->out_stride % 8) {
    errf(err, errlen, "row strides %lld %lld: each must hold its row and be a multiple of 8 elements", (long long)a->q_stride, (long long)a->out_stride);
    return 1;
  }
  if (!aligned16(a->q) || !aligned16(a->out)) { errf(err, errlen, "q or out does not start on a 16-byte boundary"); return 1; }
  if (a->T > 0) {
    const size_t T1 = static_cast<size_t>(a->T) - 1;
    if (overlap(a->out, (T1 * a->out_stride + nq) * (a->out_type == T_F32 ? 4 : 2), a->q, (T1 * a->q_stride + nq) * 2)) { errf(err, errlen, "out overlaps q"); return 1; }
  }
  return 0;
}

}  // namespace
}  // namespace clb

using namespace clb;

extern "C" size_t clb200_attention_work(clb200_ctx *c, const clb200_kv *kv, const clb200_attn *a) {
  char err[8];
  if (!c || check(kv, a, err, sizeof err)) return 0;
  return attn_plan(c->sms, *kv, *a).total;
}

extern "C" int clb200_attention(clb200_ctx *c, const clb200_kv *kv, const clb200_attn *a, void *stream, char *err, size_t errlen) {
  if (check(kv, a, err, errlen)) return 1;
  if (!c) { errf(err, errlen, "no context"); return 1; }
  if (a->T == 0 || kv->n_seq == 0) return 0;
  const AttnPlan p = attn_plan(c->sms, *kv, *a);
  if (!a->work || a->work_bytes < p.total || (reinterpret_cast<uintptr_t>(a->work) & 255)) {
    errf(err, errlen, "the workspace is %zu bytes at %p: it must be %zu bytes (clb200_attention_work) on a 256-byte boundary", a->work ? a->work_bytes : 0,
         a->work, p.total);
    return 1;
  }
  const OnDevice on(c->device);
  cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : c->stream;
  const bool f32 = a->out_type == T_F32;
  uint8_t *w = static_cast<uint8_t *>(a->work);
  for (int s0 = 0; s0 < kv->n_seq; s0 += ATTN_MAX_SEQ) {
    AttnArgs g{};
    g.kv = *kv;
    g.kv.table += static_cast<int64_t>(s0) * kv->table_stride;
    g.kv.q_start += s0;
    g.kv.kv_len += s0;
    g.kv.n_seq = std::min(kv->n_seq - s0, ATTN_MAX_SEQ);
    g.a = *a;
    g.a.window = std::min(a->window, 1 << 30);
    g.a.sinks = std::min(a->sinks, 1 << 30);
    g.err = c->small;
    g.group = a->n_head / kv->n_kv;
    g.group_inv = (65536u + g.group - 1) / g.group;
    g.page_shift = (kv->page_size & (kv->page_size - 1)) ? -1 : __builtin_ctz(kv->page_size);
    g.rows = p.rows;
    g.tpi = p.tpi;
    g.nc = p.nc;
    g.min_run = p.rows <= 32 ? 1 : 2;
    g.lead = p.rows <= 32 ? 3 : 2;   // (200 short sequences 40.0 us, 40.4 with 4; 64 of 32 heads over 32: 116, 122 with 2)
    g.piece_o = reinterpret_cast<float *>(w);
    g.piece_ml = reinterpret_cast<float2 *>(w + p.off_ml);
    g.joins = reinterpret_cast<int4 *>(w + p.off_joins);
    cudaError_t e;
    if (kv->type == T_F16) e = f32 ? launch_hd<__half, float>(g, st) : launch_hd<__half, __half>(g, st);
    else e = f32 ? launch_hd<__nv_bfloat16, float>(g, st) : launch_hd<__nv_bfloat16, __nv_bfloat16>(g, st);
    CUDA_OR(e, "launching the attention");
  }
  return 0;
}
