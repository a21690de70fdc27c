// clb200_qk_rope: norms of queries and keys, rotation by position, and the store of keys and values into a paged cache, one
// pass over the new tokens' rows.
#include <algorithm>

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

// Eight consecutive elements as floats, and eight floats rounded to the cache's type.
template <typename S>
CLB_DEV void load8(const S *p, float (&x)[8]) {
  if constexpr (sizeof(S) == 4) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    const S *h = reinterpret_cast<const S *>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(h[i]);
  }
}
template <typename C>
CLB_DEV void store8(C *p, const float (&x)[8]) {
  uint4 v;
  C *h = reinterpret_cast<C *>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = from_f32<C>(x[i]);
  *reinterpret_cast<uint4 *>(p) = v;
}

// One CTA per token. A head is held by HD / 8 lanes, eight consecutive elements each, so a warp takes 32 / (HD / 8) heads at
// a time and a lane's rotary row and head weights stay the same from head to head.
template <typename S, typename C, int HD>
__global__ void __launch_bounds__(QT) qk_rope_kernel(const QkArgs g) {
  constexpr int LPH = HD / 8, HPW = 32 / LPH;   // lanes per head, heads per warp
  __shared__ float red[2][QW];
  const clb200_qk &a = g.a;
  const clb200_kv &kv = g.kv;
  const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (row < kv.q_start[0] || row >= kv.q_start[kv.n_seq]) return;   // a row behind the last sequence
  const int s = seq_of_row(kv.q_start, kv.n_seq, row);
  const int pos = kv.kv_len[s] - kv.q_start[s + 1] + row;
  if (pos < 0 || pos >= a.n_pos) {
    if (threadIdx.x == 0) set_error(g.err, ERR_BAD_ROWS);
    return;
  }
  const int H = a.n_head, KV = kv.n_kv, li = lane % LPH;   // li: the lane's place in its head
  const S *q = static_cast<const S *>(a.q) + row * a.q_stride, *k = static_cast<const S *>(a.k) + row * a.k_stride;
  const S *v = static_cast<const S *>(a.v) + row * a.v_stride;
  float qs = 1.f, ks = 1.f;
  if (a.norm == CLB200_QK_NORM_ROW) {
    float sq = 0.f, sk = 0.f, x[8];
    for (int i = threadIdx.x; i < H * LPH; i += QT) {
      load8(q + 8 * i, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = fmaf(x[e], x[e], sq);
    }
    for (int i = threadIdx.x; i < KV * LPH; i += QT) {
      load8(k + 8 * i, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) sk = fmaf(x[e], x[e], sk);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { sq += __shfl_xor_sync(FULL_MASK, sq, o); sk += __shfl_xor_sync(FULL_MASK, sk, o); }
    if (lane == 0) { red[0][warp] = sq; red[1][warp] = sk; }
    __syncthreads();
    sq = sk = 0.f;
    for (int w = 0; w < QW; ++w) { sq += red[0][w]; sk += red[1][w]; }
    qs = 1.0f / sqrtf(sq / static_cast<float>(H * HD) + a.eps);
    ks = 1.0f / sqrtf(sk / static_cast<float>(KV * HD) + a.eps);
  }
  const int page = page_of(kv, s, pos, g.err);
  const int64_t slot = page * kv.page_stride + (pos % kv.page_size) * kv.slot_stride;
  // the lane's cosines and sines: its elements' pairs are (i, i + HD / 2), or (2i, 2i + 1) inside the lane
  const float *cs = a.rope + static_cast<int64_t>(pos) * HD;
  float c[8], n[8];
  if (a.pairs) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { c[e] = cs[4 * li + e]; n[e] = cs[HD / 2 + 4 * li + e]; }
  } else {
    load8(cs + 8 * (li % (LPH / 2)), c);
    load8(cs + HD / 2 + 8 * (li % (LPH / 2)), n);
  }
  const int hh = lane / LPH;
  for (int h0 = warp * HPW; h0 < H + KV; h0 += QW * HPW) {
    const int h = h0 + hh;
    const bool live = h < H + KV, isk = h >= H;
    const int head = isk ? h - H : h;
    float x[8];
    if (live) load8((isk ? k : q) + head * HD + 8 * li, x);
    else
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
    if (a.norm != CLB200_QK_NORM_NONE) {
      float scale = isk ? ks : qs;
      if (a.norm == CLB200_QK_NORM_HEAD) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(FULL_MASK, ss, o);
        scale = 1.0f / sqrtf(ss * (1.0f / HD) + a.eps);
      }
      if (live) {
        const float *wp = (isk ? a.k_norm : a.q_norm) + (a.norm == CLB200_QK_NORM_ROW ? head * HD : 0) + 8 * li;
        float w[8];
        load8(wp, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * scale * w[e];
      }
    }
    float y[8];
    if (a.pairs) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[2 * e] = fmaf(x[2 * e], c[e], -(x[2 * e + 1] * n[e]));
        y[2 * e + 1] = fmaf(x[2 * e], n[e], x[2 * e + 1] * c[e]);
      }
    } else {
      const bool hi = li >= LPH / 2;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float o = __shfl_xor_sync(FULL_MASK, x[e], LPH / 2);
        y[e] = hi ? fmaf(o, n[e], x[e] * c[e]) : fmaf(x[e], c[e], -(o * n[e]));
      }
    }
    if (!live) continue;
    if (!isk) store8(static_cast<C *>(a.out) + row * a.out_stride + head * HD + 8 * li, y);
    else if (page >= 0) store8(static_cast<C *>(kv.k) + slot + head * kv.head_stride + 8 * li, y);
  }
  if (page >= 0)
    for (int i = threadIdx.x; i < KV * LPH; i += QT) {
      float x[8];
      load8(v + 8 * i, x);
      store8(static_cast<C *>(kv.v) + slot + (i / LPH) * kv.head_stride + 8 * (i % LPH), x);
    }
}

template <typename S, typename C>
void launch_hd(const QkArgs &g, cudaStream_t st) {
  switch (g.kv.head_dim) {
    case 64: qk_rope_kernel<S, C, 64><<<g.a.T, QT, 0, st>>>(g); break;
    case 128: qk_rope_kernel<S, C, 128><<<g.a.T, QT, 0, st>>>(g); break;
    default: qk_rope_kernel<S, C, 256><<<g.a.T, QT, 0, st>>>(g); break;
  }
}

int check(const clb200_kv *kv, const clb200_qk *a, char *err, size_t errlen) {
  if (!kv || !a) { errf(err, errlen, "no cache or arguments"); return 1; }
  if (check_kv(kv, err, errlen)) return 1;
  if (a->T < 0 || a->n_head < 1 || a->n_head > 1024) { errf(err, errlen, "%d rows of %d query heads: out of range", a->T, a->n_head); return 1; }
  if (a->src_type != T_F32 && a->src_type != kv->type) { errf(err, errlen, "q, k and v are %s: they must be F32 or the cache's type", type_name(a->src_type)); return 1; }
  if (!a->q || !a->k || !a->v || !a->out || !a->rope) { errf(err, errlen, "a buffer is missing"); return 1; }
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
  if (static_cast<int64_t>(kv->table_width) * kv->page_size > INT32_MAX) { errf(err, errlen, "a table of %d pages of %d slots: positions must fit 31 bits", kv->table_width, kv->page_size); return 1; }
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
    if (f32) launch_hd<float, __half>(g, st);
    else launch_hd<__half, __half>(g, st);
  } else {
    if (f32) launch_hd<float, __nv_bfloat16>(g, st);
    else launch_hd<__nv_bfloat16, __nv_bfloat16>(g, st);
  }
  CUDA_OR(cudaGetLastError(), "launching the rotation");
  return 0;
}
