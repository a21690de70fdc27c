// clb200_attention: attention of chunks of new tokens over a paged key/value cache.
#include <algorithm>

#include "ctx.cuh"
#include "serve.cuh"

namespace clb {
namespace {

constexpr int AT = 128, AW = AT / 32;

struct AttnArgs {
  clb200_kv kv;
  clb200_attn a;
  int *err;
};

// One CTA per (row, query head): warp w takes every AW-th visible position, a lane HD / 32 elements of the head, with a
// running maximum and sum per warp; the warps' states are joined at the end.
template <typename C, typename O, int HD>
__global__ void __launch_bounds__(AT) attn_plain_kernel(const AttnArgs g) {
  constexpr int EPL = HD / 32;
  __shared__ float sm[AW], sl[AW], so[AW][HD];
  const clb200_attn &a = g.a;
  const clb200_kv &kv = g.kv;
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (row < kv.q_start[0] || row >= kv.q_start[kv.n_seq]) return;
  const int s = seq_of_row(kv.q_start, kv.n_seq, row);
  if (kv.q_start[s + 1] - kv.q_start[s] > a.max_q) {
    if (threadIdx.x == 0) set_error(g.err, ERR_BAD_ROWS);
    return;
  }
  const int pos = kv.kv_len[s] - kv.q_start[s + 1] + row;
  const int n = min(pos, kv.kv_len[s] - 1) + 1;
  const int kh = h / (a.n_head / kv.n_kv);
  float q[EPL], o[EPL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    q[e] = to_f32(static_cast<const C *>(a.q)[row * a.q_stride + h * HD + lane * EPL + e]);
    o[e] = 0.f;
  }
  for (int j = warp; j < n; j += AW) {
    if (a.window > 0 && j <= pos - a.window && j >= a.sinks) continue;
    const int page = page_of(kv, s, j, g.err);
    if (page < 0) continue;
    const int64_t at = page * kv.page_stride + (j % kv.page_size) * kv.slot_stride + kh * kv.head_stride + lane * EPL;
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) d = fmaf(q[e], to_f32(static_cast<const C *>(kv.k)[at + e]), d);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) d += __shfl_xor_sync(FULL_MASK, d, i);
    d *= a.scale;
    const float mn = fmaxf(m, d), f = m == -INFINITY ? 0.f : expf(m - mn), p = mn == -INFINITY ? 0.f : expf(d - mn);
    l = fmaf(l, f, p);
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] = fmaf(o[e], f, p * to_f32(static_cast<const C *>(kv.v)[at + e]));
    m = mn;
  }
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
  for (int e = 0; e < EPL; ++e) so[warp][lane * EPL + e] = o[e];
  __syncthreads();
  float mm = -INFINITY, ll = 0.f;
  for (int w = 0; w < AW; ++w) mm = fmaxf(mm, sm[w]);
  float f[AW];
  for (int w = 0; w < AW; ++w) { f[w] = sm[w] == -INFINITY ? 0.f : expf(sm[w] - mm); ll = fmaf(f[w], sl[w], ll); }
  for (int d = threadIdx.x; d < HD; d += AT) {
    float v = 0.f;
    for (int w = 0; w < AW; ++w) v = fmaf(f[w], so[w][d], v);
    static_cast<O *>(a.out)[row * a.out_stride + h * HD + d] = from_f32<O>(ll > 0.f ? v / ll : 0.f);
  }
}

template <typename C, typename O>
void launch_hd(const AttnArgs &g, cudaStream_t st) {
  const dim3 grid(g.a.T, g.a.n_head);
  switch (g.kv.head_dim) {
    case 64: attn_plain_kernel<C, O, 64><<<grid, AT, 0, st>>>(g); break;
    case 128: attn_plain_kernel<C, O, 128><<<grid, AT, 0, st>>>(g); break;
    default: attn_plain_kernel<C, O, 256><<<grid, AT, 0, st>>>(g); break;
  }
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
  if (!a->q || !a->out) { errf(err, errlen, "a buffer is missing"); return 1; }
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
  if (!c || !kv || !a) return 0;
  return 0;
}

extern "C" int clb200_attention(clb200_ctx *c, const clb200_kv *kv, const clb200_attn *a, void *stream, char *err, size_t errlen) {
  if (check(kv, a, err, errlen)) return 1;
  if (!c) { errf(err, errlen, "no context"); return 1; }
  if (a->T == 0 || kv->n_seq == 0) return 0;
  const OnDevice on(c->device);
  const AttnArgs g{*kv, *a, c->small};
  cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : c->stream;
  const bool f32 = a->out_type == T_F32;
  if (kv->type == T_F16) {
    if (f32) launch_hd<__half, float>(g, st);
    else launch_hd<__half, __half>(g, st);
  } else {
    if (f32) launch_hd<__nv_bfloat16, float>(g, st);
    else launch_hd<__nv_bfloat16, __nv_bfloat16>(g, st);
  }
  CUDA_OR(cudaGetLastError(), "launching the attention");
  return 0;
}
