// clb200_attention for many rows per key/value head: tcgen05 tiles (accumulators in TMEM) fed by TMA from the pages.
//
// An item's rows (new tokens x the group's query heads) fill up to two tiles of 128 rows, the streams; both use every key and
// value tile of N positions that is loaded. A CTA per SM walks its run of tiles (attn.cuh) with
//   warps of softmax group w (128 threads, a row each): load the stream's queries into shared memory; per tile read their row
//           of the scores S_w from TMEM, mask, take the exponentials against the row's running maximum, keep its sum, and
//           write the probabilities back over S_w as the operand P_w; at the end of the item read O_w and store it;
//   one warp (TMA): the item's key and value tiles through a ring of stages, a box per page piece; positions at or past the
//           sequence's end come from outside the tensor, as zeros, except inside the last box;
//   one warp (MMA): S_w = Q_w K^T (both operands in shared memory), O_w += P_w V (P_w from TMEM). While group 0 works on its
//           scores the tensor cores run the other stream's products.
// The maximum that scales a row's sums is only moved when the row's maximum has grown by more than 2^8 (the probabilities then
// reach 2^8 at most, far inside fp16 and fp32), so rescaling O_w, a round trip through the registers, is rare.
// The values of positions past the sequence's end inside the last box may be anything, and 0 x NaN is NaN: the MMA warp zeroes
// their rows in shared memory. Every wait is bounded; one that runs out sets the error word.
#include <cuda.h>

#include <algorithm>
#include <numeric>

#include "attn.cuh"
#include "ctx.cuh"
#include "tcgen05.cuh"

namespace clb {
namespace {

template <int HD>
struct TcAttn {
  static constexpr int STREAMS = HD == 256 ? 1 : 2;          // O of 256 columns leaves room for one stream
  static constexpr int N = HD == 256 ? 64 : 128;             // positions per tile
  static constexpr int THREADS = 128 * (STREAMS + 1);
  static constexpr uint32_t Q_TILE = 128 * HD * 2, STAGE = N * HD * 2;
  static constexpr int STAGES = HD == 64 ? 10 : 5;
  static constexpr int N_BARS = 2 * STAGES + 4 * STREAMS + 1;
  static constexpr uint32_t SMEM = 1024 + STREAMS * Q_TILE + STAGES * STAGE + 8 * N_BARS + 16;
  static constexpr uint32_t S_COL = 0, O_COL = 256;          // S_w at 128 w (P_w over its first half), O_w at 256 + HD w
  static_assert(SMEM <= 232448, "shared memory budget");
  static_assert((ATTN_MAX_SEQ + 1) * 8 <= STAGES * STAGE, "the prefix sums fit the ring");
};

CLB_DEV void tma_load_4d(void *dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
               : "memory");
}

template <typename C>
CLB_DEV uint32_t pack_pair(float a, float b) {   // a in the low half
  if constexpr (__is_same(C, __half)) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}

template <typename C, typename O, int HD>
__global__ void __launch_bounds__(TcAttn<HD>::THREADS, 1)
    attn_tc_kernel(const AttnArgs g, const int box, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using S = TcAttn<HD>;
  constexpr int N = S::N, ST = S::STREAMS;
  constexpr bool BF16 = __is_same(C, __nv_bfloat16);
  extern __shared__ uint8_t raw[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t *ring = sm + ST * S::Q_TILE;
  uint64_t *kv_full = reinterpret_cast<uint64_t *>(ring + S::STAGES * S::STAGE), *kv_free = kv_full + S::STAGES;
  uint64_t *q_full = kv_free + S::STAGES, *s_full = q_full + ST, *p_full = s_full + ST, *o_full = p_full + ST, *mma_done = o_full + ST;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mma_done + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
  const clb200_attn &a = g.a;
  const clb200_kv &kv = g.kv;
  const int tps = 128 / g.group;   // new tokens per stream

  AttnRun<N> run;
  run.init(g, reinterpret_cast<int64_t *>(ring), cta);
  if (tid == 0) {
    g.joins[cta] = make_int4(0, 0, 0, 0);
    for (int i = 0; i < S::STAGES; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_free[i], 1); }
    for (int w = 0; w < ST; ++w) { mbar_init(&q_full[w], 4); mbar_init(&s_full[w], 1); mbar_init(&p_full[w], 4); mbar_init(&o_full[w], 1); }
    mbar_init(mma_done, 1);
    fence_barrier_init();
  }
  fence_proxy_async();   // the ring held the prefix sums: the copies that fill it come after them
  if (warp == 0) tc::tmem_alloc(tmem_slot, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp >= 4 * ST) {
    if constexpr (ST == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 4 * ST) {   // ---- TMA
      uint32_t cnt = 0;
      const int boxes = N / box;
      auto load = [&](const CUtensorMap &map, const AttnSeq &q, int s, int head, int tile) -> bool {
        const uint32_t st = cnt % S::STAGES;
        if (cnt >= S::STAGES && !mbar_wait_bounded(&kv_free[st], (cnt / S::STAGES - 1) & 1)) return false;
        if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], S::STAGE);
        __syncwarp();
        if (lane < boxes) {
          const int pos = tile * N + lane * box;
          int page = kv.n_pages, slot = 0;   // outside the tensor: zeros
          if (pos < q.kv) {
            page = page_of(kv, s, pos, g.err);
            if (page < 0) page = kv.n_pages;
            slot = pos % kv.page_size;
          }
          uint8_t *dst = ring + st * S::STAGE + lane * box * 128;
#pragma unroll
          for (int cb = 0; cb < HD / 64; ++cb) tma_load_4d(dst + cb * N * 128, &map, 64 * cb, head, slot, page, &kv_full[st]);
        }
        ++cnt;
        return true;
      };
      while (ok && run.more()) {
        const AttnSpan span = attn_span<N>(g, run.q, run.qt);
        const int n = run.tiles(span), i0 = run.i0;
        ok = load(map_k, run.q, run.s, run.head, span.tile(i0));
        for (int j = 0; ok && j < n; ++j) {
          if (j + 1 < n) ok = load(map_k, run.q, run.s, run.head, span.tile(i0 + j + 1));
          if (ok) ok = load(map_v, run.q, run.s, run.head, span.tile(i0 + j));
        }
        run.advance(g, n);
      }
      // every copy issued has landed before the CTA exits (already so unless a wait gave up)
      for (uint32_t v = cnt > S::STAGES ? cnt - S::STAGES : 0; v < cnt; ++v)
        if (!mbar_wait_bounded(&kv_full[v % S::STAGES], (v / S::STAGES) & 1)) ok = false;
    } else if (warp == 4 * ST + 1) {   // ---- MMA
      constexpr uint32_t ID_S = tc::idesc_half(BF16, false, 128, N), ID_O = tc::idesc_half(BF16, true, 128, HD);
      uint32_t cnt = 0, items[ST] = {}, tiles[ST] = {};   // stages, items and tiles consumed
      auto scores = [&](int w, uint32_t st) {             // S_w = Q_w K^T; lane 0
        const uint64_t qd = tc::sw128_desc(smem_addr(sm + w * S::Q_TILE)), kd = tc::sw128_desc(smem_addr(ring + st * S::STAGE));
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          tc::mma_f16(tmem + S::S_COL + 128 * w, qd + (kk / 4) * (128 * 128 / 16) + 2 * (kk % 4), kd + (kk / 4) * (N * 128 / 16) + 2 * (kk % 4), ID_S, kk != 0);
        tc::commit(&s_full[w]);
      };
      while (ok && run.more()) {
        const AttnSeq q = run.q;
        const AttnSpan span = attn_span<N>(g, q, run.qt);
        const int n = run.tiles(span), i0 = run.i0;
        const int live = ST == 2 && q.nq - run.qt * g.tpi > tps ? 2 : 1;   // streams that have rows
        const uint32_t k0 = cnt++ % S::STAGES;
        if (!mbar_wait_bounded(&kv_full[k0], ((cnt - 1) / S::STAGES) & 1)) { ok = false; break; }
        for (int w = 0; ok && w < live; ++w) {
          if (!mbar_wait_bounded(&q_full[w], items[w]++ & 1)) ok = false;
          tc::fence_after_sync();
          if (ok && lane == 0) scores(w, k0);
        }
        if (!ok) break;
        if (lane == 0) tc::commit(&kv_free[k0]);
        for (int j = 0; j < n; ++j) {
          uint32_t ks = 0;
          if (j + 1 < n) {
            ks = cnt++ % S::STAGES;
            if (!mbar_wait_bounded(&kv_full[ks], ((cnt - 1) / S::STAGES) & 1)) { ok = false; break; }
          }
          const uint32_t vs = cnt++ % S::STAGES;
          if (!mbar_wait_bounded(&kv_full[vs], ((cnt - 1) / S::STAGES) & 1)) { ok = false; break; }
          const int left = q.kv - span.tile(i0 + j) * N;   // rows of the tile that are the sequence's
          if (left < N) {
            for (int i = lane; i < (N - max(left, 0)) * 8 * (HD / 64); i += 32) {
              const int c = i & 7, cb = (i >> 3) % (HD / 64), r = max(left, 0) + (i >> 3) / (HD / 64);
              *reinterpret_cast<uint4 *>(ring + vs * S::STAGE + cb * N * 128 + r * 128 + 16 * c) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();
            __syncwarp();
          }
          const uint64_t vd = tc::sw128_desc_mn(smem_addr(ring + vs * S::STAGE), N * 128);
          for (int w = 0; w < live; ++w) {
            if (!mbar_wait_bounded(&p_full[w], tiles[w]++ & 1)) { ok = false; break; }
            tc::fence_after_sync();
            if (lane == 0) {
#pragma unroll
              for (int kk = 0; kk < N / 16; ++kk)
                tc::mma_f16_ts(tmem + S::O_COL + HD * w, tmem + S::S_COL + 128 * w + 8 * kk, vd + 128 * kk, ID_O, j != 0 || kk != 0);
              if (j + 1 < n) scores(w, ks);
              else tc::commit(&o_full[w]);
            }
          }
          if (!ok) break;
          if (lane == 0) {
            tc::commit(&kv_free[vs]);
            if (j + 1 < n) tc::commit(&kv_free[ks]);
          }
        }
        run.advance(g, n);
      }
      if (lane == 0) {
        tc::commit(mma_done);   // the TMEM is released only after every MMA issued has completed
        if (!mbar_wait_bounded(mma_done, 0)) ok = false;
      }
    }
  } else {   // ---- softmax group w, a row per thread
    if constexpr (ST == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int w = warp >> 2, r = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_col = tmem + lanes + S::S_COL + 128 * w, o_col = tmem + lanes + S::O_COL + HD * w;
    const float sc = a.scale * LOG2E;
    uint8_t *qt_sm = sm + w * S::Q_TILE;
    uint32_t items = 0, tiles = 0;
    auto mine = [&]() { return w == 0 || run.q.nq - run.qt * g.tpi > tps; };   // whether the item has rows in this stream
    auto load_q = [&]() {
      const int t0 = run.qt * g.tpi + w * tps;
      for (int i = r; i < 128 * (HD / 8); i += 128) {
        const int row = i / (HD / 8), c = i % (HD / 8), t = t0 + row / g.group;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < tps * g.group && t < run.q.nq)
          v = *reinterpret_cast<const uint4 *>(static_cast<const C *>(a.q) + (run.q.row + t) * a.q_stride + (run.head * g.group + row % g.group) * HD + 8 * c);
        *reinterpret_cast<uint4 *>(qt_sm + (c >> 3) * (128 * 128) + tc::sw128_chunk(row, c & 7)) = v;
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[w]);
    };
    while (run.more() && !mine()) run.advance(g, run.tiles(attn_span<N>(g, run.q, run.qt)));
    if (run.more()) load_q();
    while (ok && run.more()) {
      const AttnSeq q = run.q;
      const AttnSpan span = attn_span<N>(g, q, run.qt);
      const int n = run.tiles(span), i0 = run.i0, head = run.head, t0 = run.qt * g.tpi + w * tps, t = t0 + r / g.group;
      const bool whole = n == span.nt, row_live = r < tps * g.group && t < q.nq;
      const int first = span.lo + w * tps;            // position of the stream's first token
      const int pos = first + r / g.group;
      float m = -INFINITY;
      float2 l0 = make_float2(0.f, 0.f), l1 = l0;
      for (int j = 0; j < n; ++j) {
        if (!mbar_wait_bounded(&s_full[w], tiles++ & 1)) { ok = false; break; }
        tc::fence_after_sync();
        uint32_t xr[N];
#pragma unroll
        for (int c = 0; c < N / 32; ++c) tc::ld_x32_async(s_col + 32 * c, xr + 32 * c);
#pragma unroll
        for (int c = 0; c < N / 32; ++c) tc::wait_ld_x32(xr + 32 * c);
        float *x = reinterpret_cast<float *>(xr);
        const int p0 = span.tile(i0 + j) * N;
        // some row of the stream does not see the whole tile
        if (p0 + N - 1 > first || (a.window > 0 && p0 <= span.hi - a.window && p0 + N - 1 >= a.sinks)) {
          const int hi = pos - p0, lo = a.window > 0 ? pos - a.window - p0 : -1, sk = a.window > 0 ? a.sinks - p0 : 0;
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (i > hi || (i <= lo && i >= sk)) x[i] = -INFINITY;
        }
        float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int i = 4; i < N; ++i) mx[i & 3] = fmaxf(mx[i & 3], x[i]);
        const float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
        if (__any_sync(FULL_MASK, mn > m + 8.0f)) {   // also where m is still -infinity
          const float mb = fmaxf(m, mn), f = m == -INFINITY ? 0.f : exp2_approx(m - mb);
          m = mb;
          l0.x *= f; l0.y *= f; l1.x *= f; l1.y *= f;
          if (j > 0) {   // the products before this tile's scores are complete: O_w is at rest
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t o[32];
              tc::ld_x32_async(o_col + 32 * c, o);
              tc::wait_ld_x32(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tc::st_x32(o_col + 32 * c, o);
            }
          }
        }
        const float z = m == -INFINITY ? 0.f : m;
        const float2 sc2 = make_float2(sc, sc), nz = make_float2(-z, -z);
        // the probabilities go into the product in the cache's type (its operands share a type); their sum stays fp32
#pragma unroll
        for (int h = 0; h < N / 64; ++h) {
          uint32_t p[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float2 v = ffma2(make_float2(x[64 * h + 2 * i], x[64 * h + 2 * i + 1]), sc2, nz);
            v.x = exp2_approx(v.x);
            v.y = exp2_approx(v.y);
            if (i & 1) l1 = fadd2(l1, v);
            else l0 = fadd2(l0, v);
            p[i] = pack_pair<C>(v.x, v.y);
          }
          tc::st_x32(s_col + 32 * h, p);
        }
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[w]);
      }
      if (!ok) break;
      if (i0 == 0 && !whole && tid == 0) g.joins[cta] = make_int4(run.s, head, run.qt, run.pieces(span.nt - n));
      // the next item's queries: every product that reads this item's is complete (its last scores have been read)
      run.advance(g, n);
      while (run.more() && !mine()) run.advance(g, run.tiles(attn_span<N>(g, run.q, run.qt)));
      if (run.more()) load_q();
      else grid_launch_dependents();
      if (!mbar_wait_bounded(&o_full[w], items++ & 1)) { ok = false; break; }
      tc::fence_after_sync();
      const float l = (l0.x + l0.y) + (l1.x + l1.y), inv = l > 0.f ? 1.0f / l : 0.f;
      const int64_t piece = static_cast<int64_t>(2 * cta + (i0 == 0 ? 1 : 0)) * g.rows + w * tps * g.group + r;
      O *dst = static_cast<O *>(a.out) + (row_live ? (q.row + t) * a.out_stride + (head * g.group + r % g.group) * HD : 0);
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        tc::ld_x32_async(o_col + 32 * c, o);
        tc::wait_ld_x32(o);
        if (!row_live) continue;
        const float *v = reinterpret_cast<const float *>(o);
        if (whole) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) store4<O>(dst + 32 * c + i, make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]), inv);
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4 *>(g.piece_o + piece * HD + 32 * c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
      if (!whole && row_live) g.piece_ml[piece] = make_float2(m, l);
      tc::fence_before_sync();
    }
  }
  if (!ok) set_error(g.err, ERR_WAIT_COPY);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 0) tc::tmem_dealloc(tmem, 512);
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
  static EncodeTiled fn = nullptr;
  if (!fn) {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && p) fn = reinterpret_cast<EncodeTiled>(p);
  }
  return fn;
}

// The pages as a tensor (element, head, slot, page): boxes of 64 elements of one head by `box` slots of one page, 128-byte
// swizzle, zeros outside.
bool encode_pages(CUtensorMap *m, const clb200_kv &kv, const void *base, int box) {
  const EncodeTiled fn = encoder();
  if (!fn) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(kv.head_dim), static_cast<cuuint64_t>(kv.n_kv), static_cast<cuuint64_t>(kv.page_size),
                              static_cast<cuuint64_t>(kv.n_pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(kv.n_kv > 1 ? kv.head_stride : kv.head_dim) * 2, static_cast<cuuint64_t>(kv.slot_stride) * 2,
                                 static_cast<cuuint64_t>(kv.n_pages > 1 ? kv.page_stride : kv.head_dim) * 2};
  const cuuint32_t boxes[4] = {64, 1, static_cast<cuuint32_t>(box), 1}, estr[4] = {1, 1, 1, 1};
  return fn(m, kv.type == T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides, boxes,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename C, typename O, int HD>
cudaError_t launch(const AttnArgs &g, cudaStream_t st) {
  using S = TcAttn<HD>;
  static bool done[64] = {};
  const cudaError_t e = allow_smem(attn_tc_kernel<C, O, HD>, S::SMEM, done);
  if (e != cudaSuccess) return e;
  const int box = std::gcd(g.kv.page_size, S::N);
  CUtensorMap mk, mv;
  if (!encode_pages(&mk, g.kv, g.kv.k, box) || !encode_pages(&mv, g.kv, g.kv.v, box)) return cudaErrorInvalidValue;
  attn_tc_kernel<C, O, HD><<<g.nc, S::THREADS, S::SMEM, st>>>(g, box, mk, mv);
  return cudaGetLastError();
}

template <typename C, typename O>
cudaError_t launch_hd(const AttnArgs &g, cudaStream_t st) {
  switch (g.kv.head_dim) {
    case 64: return launch<C, O, 64>(g, st);
    case 128: return launch<C, O, 128>(g, st);
    default: return launch<C, O, 256>(g, st);
  }
}

}  // namespace

cudaError_t launch_attn_tc(const AttnArgs &g, cudaStream_t st) {
  const bool f32 = g.a.out_type == T_F32;
  if (g.kv.type == T_F16) return f32 ? launch_hd<__half, float>(g, st) : launch_hd<__half, __half>(g, st);
  return f32 ? launch_hd<__nv_bfloat16, float>(g, st) : launch_hd<__nv_bfloat16, __nv_bfloat16>(g, st);
}

}  // namespace clb
