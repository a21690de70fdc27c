// clb200_qk_rope: norms of queries and keys, rotation by position, and the store of keys and values into a paged cache, one
// pass over the new tokens' rows.
#include <algorithm>
#include <type_traits>

#include "ctx.cuh"
#include "serve.cuh"

namespace clb {
namespace {

constexpr int QT = 256;         // threads of a CTA
constexpr int QW = QT / 32;

struct QkArgs {
  clb200_kv kv;
  clb200_qk a;
  int *err;
};

// Four consecutive elements as they lie in memory, as floats, and rounded to the cache's type.
template <typename S>
struct Raw4 {
  using W = typename std::conditional<sizeof(S) == 4, uint4, uint2>::type;
  W v;
  CLB_DEV void load(const S *p) { v = *reinterpret_cast<const W *>(p); }
  CLB_DEV void get(float *x) const {
    const S *h = reinterpret_cast<const S *>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f32(h[i]);
  }
};
CLB_DEV void load4(const float *p, float *x) {
  const float4 v = *reinterpret_cast<const float4 *>(p);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
template <typename C>
CLB_DEV void put4(C *p, const float *x) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<C>(x[0], x[1]), pack2<C>(x[2], x[3]));
}

// One token by WARPS warps (a CTA's eight, or one of them). A head is held by HD / 8 lanes, each four consecutive elements of its
// first half and the same four of its second, so both rotations stay inside the lane, and a lane's rotary values and head
// weights are the same from head to head; a warp takes 32 / (HD / 8) heads at a time.
// The bound is memory: every element is read and written once. What stands in its way is latency, since where a token's few
// kilobytes go hangs on a chain of look-ups (the sequence by bisection, its length, the page). The queries, whose place depends
// on the row alone, are requested before it, HOLD rounds of heads a warp. With a CTA per token the chain is a token's whole
// time; a warp per token has as many tokens in flight as an SM has warps, and pays off once there are tokens for them.
// At 5 ragged prompts of 64 + 4 + 4 heads of 128, bf16 (231 MB): 46 us with a warp per token (5.0 TB/s), 70 with a CTA; 68 while
// a lane held eight consecutive elements, half of whose partners came by shuffles (192 instructions a round, the issue rate then
// being the limit).
template <typename S, typename C, int HD, int WARPS>
__global__ void __launch_bounds__(QT, WARPS == 1 ? 3 : 1) qk_rope_kernel(const QkArgs g) {
  constexpr int LPH = HD / 8, HPW = 32 / LPH, ROUND = WARPS * HPW, HALF = HD / 2;   // lanes per head, heads per warp, heads per round
  constexpr int HOLD = sizeof(S) == 4 ? 3 : 4;                                       // rounds whose loads are in flight at once
  __shared__ float red[2][QW];
  const clb200_qk &a = g.a;
  const clb200_kv &kv = g.kv;
  const int lane = threadIdx.x & 31, warp = WARPS == 1 ? 0 : threadIdx.x >> 5, part = WARPS == 1 ? lane : threadIdx.x;
  const int row = WARPS == 1 ? blockIdx.x * QW + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.T) return;
  const int H = a.n_head, KV = kv.n_kv, at = 4 * (lane % LPH), mine = warp * HPW + lane / LPH;   // the lane's elements, its first head
  const S *q = static_cast<const S *>(a.q) + row * a.q_stride + at, *k = static_cast<const S *>(a.k) + row * a.k_stride + at;
  Raw4<S> raw[HOLD][2];
  auto fetch = [&](const S *p, int h0, int n) {   // HOLD rounds of n heads from h0 on
#pragma unroll
    for (int u = 0; u < HOLD; ++u) {
      const int h = h0 + u * ROUND + mine;
      if (h < n) {
        raw[u][0].load(p + h * HD);
        raw[u][1].load(p + h * HD + HALF);
      }
    }
  };
  fetch(q, 0, H);
  if (row < kv.q_start[0] || row >= kv.q_start[kv.n_seq]) return;   // a row behind the last sequence
  const int s = seq_of_row(kv.q_start, kv.n_seq, row);
  const int pos = kv.kv_len[s] - kv.q_start[s + 1] + row;
  if (pos < 0 || pos >= a.n_pos) {
    if (part == 0) set_error(g.err, ERR_BAD_ROWS);
    return;
  }
  const int page = page_of(kv, s, pos, g.err);
  // the cosines and sines of the lane's pairs: (i, i + HALF) for its four i, or (2i, 2i + 1), two in each half
  const float *cs = a.rope + static_cast<int64_t>(pos) * HD;
  float c[4], n[4], wq[8], wk[8];
  if (a.pairs) {
    const float2 c0 = *reinterpret_cast<const float2 *>(cs + at / 2), c1 = *reinterpret_cast<const float2 *>(cs + HALF / 2 + at / 2);
    const float2 n0 = *reinterpret_cast<const float2 *>(cs + HALF + at / 2), n1 = *reinterpret_cast<const float2 *>(cs + HALF + HALF / 2 + at / 2);
    c[0] = c0.x; c[1] = c0.y; c[2] = c1.x; c[3] = c1.y;
    n[0] = n0.x; n[1] = n0.y; n[2] = n1.x; n[3] = n1.y;
  } else {
    load4(cs + at, c);
    load4(cs + HALF + at, n);
  }
  if (a.norm == CLB200_QK_NORM_HEAD) {
    load4(a.q_norm + at, wq);
    load4(a.q_norm + HALF + at, wq + 4);
    load4(a.k_norm + at, wk);
    load4(a.k_norm + HALF + at, wk + 4);
  }
  float qs = 1.f, ks = 1.f;
  if (a.norm == CLB200_QK_NORM_ROW) {
    auto squares = [&](const S *p, int heads) {
      float t = 0.f;
      for (int h0 = 0; h0 < heads; h0 += HOLD * ROUND) {
        fetch(p, h0, heads);
#pragma unroll
        for (int u = 0; u < HOLD; ++u) {
          if (h0 + u * ROUND + mine >= heads) continue;
          float x[8];
          raw[u][0].get(x);
          raw[u][1].get(x + 4);
#pragma unroll
          for (int e = 0; e < 8; ++e) t = fmaf(x[e], x[e], t);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(FULL_MASK, t, o);
      return t;
    };
    float sk = squares(k, KV), sq = squares(q, H);
    if constexpr (WARPS > 1) {
      if (lane == 0) { red[0][warp] = sq; red[1][warp] = sk; }
      __syncthreads();
      sq = sk = 0.f;
      for (int w = 0; w < WARPS; ++w) { sq += red[0][w]; sk += red[1][w]; }
    }
    qs = 1.0f / sqrtf(sq / static_cast<float>(H * HD) + a.eps);
    ks = 1.0f / sqrtf(sk / static_cast<float>(KV * HD) + a.eps);
    if (H > HOLD * ROUND) fetch(q, 0, H);   // the first rounds' registers hold the last ones
  }
  // the heads of p, HOLD rounds at a time: the first rounds are on their way already
  auto turn = [&](const S *p, int heads, const float *norm, const float (&w)[8], float scale, C *dst, int64_t dst_stride, bool store) {
    for (int h0 = 0; h0 < heads; h0 += HOLD * ROUND) {
      if (h0) fetch(p, h0, heads);
#pragma unroll
      for (int u = 0; u < HOLD; ++u) {
        if (h0 + u * ROUND + warp * HPW >= heads) break;   // none of the warp's
        const int h = h0 + u * ROUND + mine;
        float x[8], y[8];
        raw[u][0].get(x);
        raw[u][1].get(x + 4);
        if (a.norm == CLB200_QK_NORM_HEAD) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
          for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(FULL_MASK, ss, o);
          ss = rsqrtf(fmaf(ss, 1.0f / HD, a.eps));   // within 2^-22
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= ss * w[e];
        } else if (a.norm == CLB200_QK_NORM_ROW && h < heads) {
          load4(norm + h * HD + at, y);
          load4(norm + h * HD + HALF + at, y + 4);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= scale * y[e];
        }
        if (a.pairs) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[2 * e] = fmaf(x[2 * e], c[e], -(x[2 * e + 1] * n[e]));
            y[2 * e + 1] = fmaf(x[2 * e], n[e], x[2 * e + 1] * c[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[e] = fmaf(x[e], c[e], -(x[e + 4] * n[e]));
            y[e + 4] = fmaf(x[e], n[e], x[e + 4] * c[e]);
          }
        }
        if (store && h < heads) {
          put4(dst + h * dst_stride, y);
          put4(dst + h * dst_stride + HALF, y + 4);
        }
      }
    }
  };
  turn(q, H, a.q_norm, wq, qs, static_cast<C *>(a.out) + row * a.out_stride + at, HD, true);
  const int64_t slot = page * kv.page_stride + (pos % kv.page_size) * kv.slot_stride + at;
  fetch(k, 0, KV);
  turn(k, KV, a.k_norm, wk, ks, static_cast<C *>(kv.k) + slot, kv.head_stride, page >= 0);
  if (page < 0) return;
  const S *v = static_cast<const S *>(a.v) + row * a.v_stride + at;
  C *vd = static_cast<C *>(kv.v) + slot;
  for (int h0 = 0; h0 < KV; h0 += HOLD * ROUND) {
    fetch(v, h0, KV);
#pragma unroll
    for (int u = 0; u < HOLD; ++u) {
      const int h = h0 + u * ROUND + mine;
      if (h >= KV) continue;
      float x[8];
      raw[u][0].get(x);
      raw[u][1].get(x + 4);
      put4(vd + h * kv.head_stride, x);
      put4(vd + h * kv.head_stride + HALF, x + 4);
    }
  }
}

template <typename S, typename C, int HD>
void launch(const QkArgs &g, int sms, cudaStream_t st) {
  // A warp per token once CTAs of eight tokens fill the SMs. Device time, a CTA per token and a warp per token, of 32 + 4 heads of
  // 128 in fp32: 600 tokens 8.3 and 8.8 us, 900 10.4 and 9.2, 1200 15.0 and 12.6, 1500 20.8 and 14.4; 64 + 4 in bf16: 600 9.8 and
  // 13.3, 900 13.0 and 13.3, 1200 19.3 and 18.3; 16 + 16 with the norm over the row: 900 15.8 and 16.3, 1200 22.8 and 20.3; heads of
  // 256 and of 64 cross earlier (16 + 2 of 256: 900 10.4 and 8.6; 24 + 8 of 64: 300 5.7 and 5.5).
  if (g.a.T >= QW * sms) qk_rope_kernel<S, C, HD, 1><<<(g.a.T + QW - 1) / QW, QT, 0, st>>>(g);
  else qk_rope_kernel<S, C, HD, QW><<<g.a.T, QT, 0, st>>>(g);
}
template <typename S, typename C>
void launch_hd(const QkArgs &g, int sms, cudaStream_t st) {
  switch (g.kv.head_dim) {
    case 64: launch<S, C, 64>(g, sms, st); break;
    case 128: launch<S, C, 128>(g, sms, st); break;
    default: launch<S, C, 256>(g, sms, st); break;
  }
}

int check(const clb200_kv *kv, const clb200_qk *a, char *err, size_t errlen) {
  if (!kv || !a) { errf(err, errlen, "no cache or arguments"); return 1; }
  if (check_kv(kv, err, errlen)) return 1;
  if (a->T < 0 || a->n_head < 1 || a->n_head > 1024) { errf(err, errlen, "%d rows of %d query heads: out of range", a->T, a->n_head); return 1; }
  if (a->src_type != T_F32 && a->src_type != kv->type) { errf(err, errlen, "q, k and v are %s: they must be F32 or the cache's type", type_name(a->src_type)); return 1; }
  if ((a->T > 0 && (!a->q || !a->k || !a->v || !a->out)) || !a->rope) { errf(err, errlen, "a buffer is missing"); return 1; }
  if (a->norm < CLB200_QK_NORM_NONE || a->norm > CLB200_QK_NORM_HEAD) { errf(err, errlen, "norm %d: 0 (none), 1 (row) or 2 (head)", a->norm); return 1; }
  if (a->norm && (!a->q_norm || !a->k_norm)) { errf(err, errlen, "the norm's weights are missing"); return 1; }
  if (a->pairs != 0 && a->pairs != 1) { errf(err, errlen, "pairs %d: 0 or 1", a->pairs); return 1; }
  if (a->n_pos < 1) { errf(err, errlen, "a rotary table of %d positions", a->n_pos); return 1; }
  const int64_t nq = static_cast<int64_t>(a->n_head) * kv->head_dim, nk = static_cast<int64_t>(kv->n_kv) * kv->head_dim;
  if (a->q_stride < nq || a->k_stride < nk || a->v_stride < nk || a->out_stride < nq || a->q_stride % 8 || a->k_stride % 8 ||
      a->v_stride % 8 || a->out_stride % 8) {
    errf(err, errlen, "row strides %lld %lld %lld %lld: each must hold its row and be a multiple of 8 elements", (long long)a->q_stride,
         (long long)a->k_stride, (long long)a->v_stride, (long long)a->out_stride);
    return 1;
  }
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out) || !aligned16(a->rope) || !aligned16(a->q_norm) ||
      !aligned16(a->k_norm)) {
    errf(err, errlen, "a buffer does not start on a 16-byte boundary");
    return 1;
  }
  if (a->T > 0) {
    const size_t sz = a->src_type == T_F32 ? 4 : 2, T1 = static_cast<size_t>(a->T) - 1;
    const size_t on = (T1 * a->out_stride + nq) * 2;
    if (overlap(a->out, on, a->q, (T1 * a->q_stride + nq) * sz) || overlap(a->out, on, a->k, (T1 * a->k_stride + nk) * sz) ||
        overlap(a->out, on, a->v, (T1 * a->v_stride + nk) * sz)) {
      errf(err, errlen, "out overlaps an input");
      return 1;
    }
  }
  return 0;
}

}  // namespace

int check_kv(const clb200_kv *kv, char *err, size_t errlen) {
  if (kv->type != T_F16 && kv->type != T_BF16) { errf(err, errlen, "the cache is %s: it must be F16 or BF16", type_name(kv->type)); return 1; }
  if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) { errf(err, errlen, "head_dim %d: 64, 128 or 256", kv->head_dim); return 1; }
  if (kv->page_size < 16 || kv->page_size % 16 || kv->page_size > 65536) { errf(err, errlen, "page_size %d: a multiple of 16, at most 65536", kv->page_size); return 1; }
  if (kv->n_kv < 1 || kv->n_kv > 1024 || kv->n_pages < 1 || kv->n_seq < 0 || kv->n_seq > 65535 || kv->table_width < 0 || kv->table_stride < kv->table_width) {
    errf(err, errlen, "a cache of %d pages with %d heads for %d sequences, table %d x %d: out of range", kv->n_pages, kv->n_kv, kv->n_seq,
         kv->n_seq, kv->table_width);
    return 1;
  }
  if (static_cast<int64_t>(kv->table_width) * kv->page_size > (1 << 30)) { errf(err, errlen, "a table of %d pages of %d slots: at most 2^30 positions", kv->table_width, kv->page_size); return 1; }
  if (kv->page_stride < 0 || kv->slot_stride < 0 || kv->head_stride < 0 || kv->page_stride % 8 || kv->slot_stride % 8 || kv->head_stride % 8 ||
      (kv->n_kv > 1 && kv->head_stride < kv->head_dim) || kv->slot_stride < kv->head_dim || (kv->n_pages > 1 && kv->page_stride < kv->head_dim)) {
    errf(err, errlen, "cache strides %lld %lld %lld: multiples of 8 elements that keep heads, slots and pages apart", (long long)kv->page_stride,
         (long long)kv->slot_stride, (long long)kv->head_stride);
    return 1;
  }
  if (!kv->k || !kv->v || !kv->q_start || (kv->n_seq > 0 && (!kv->kv_len || (kv->table_width > 0 && !kv->table)))) { errf(err, errlen, "a buffer of the cache is missing"); return 1; }
  if (!aligned16(kv->k) || !aligned16(kv->v)) { errf(err, errlen, "k or v does not start on a 16-byte boundary"); return 1; }
  return 0;
}

}  // namespace clb

using namespace clb;

extern "C" int clb200_qk_rope(clb200_ctx *c, const clb200_kv *kv, const clb200_qk *a, void *stream, char *err, size_t errlen) {
  if (check(kv, a, err, errlen)) return 1;
  if (!c) { errf(err, errlen, "no context"); return 1; }
  if (a->T == 0 || kv->n_seq == 0) return 0;
  const OnDevice on(c->device);
  const QkArgs g{*kv, *a, c->small};
  cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : c->stream;
  const bool f32 = a->src_type == T_F32;
  if (kv->type == T_F16) {
    if (f32) launch_hd<float, __half>(g, c->sms, st);
    else launch_hd<__half, __half>(g, c->sms, st);
  } else {
    if (f32) launch_hd<float, __nv_bfloat16>(g, c->sms, st);
    else launch_hd<__nv_bfloat16, __nv_bfloat16>(g, c->sms, st);
  }
  CUDA_OR(cudaGetLastError(), "launching the rotation");
  return 0;
}
