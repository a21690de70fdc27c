// clb200_attention for many rows per key/value head: tcgen05 tiles (accumulators in TMEM) fed by TMA from the pages.
//
// An item's rows (new tokens x the group's query heads) fill up to two tiles of 128 rows, the streams; both use every key and
// value tile of N positions that is loaded. A CTA per SM walks its run of tiles (attn.cuh) with
//   softmax group w (128 threads, a row each): per tile read their row of the scores S_w from TMEM, mask, take the exponentials
//           against the row's running maximum, keep its sum, and write the probabilities back over S_w as the operand P_w; at
//           the end of the item read O_w and store it;
//   items   (one warp): walks the run and puts each item's numbers into shared memory for the others;
//   queries (one warp): a stream's queries by TMA (a box of tokens x the group's heads x 64 elements is 128-byte-swizzled rows
//           in order) once the item before has no product left that reads them;
//   keys    (one warp): the item's key and value tiles through a ring of stages, a box per page piece; positions at or past the
//           sequence's end come from outside the tensor, as zeros, except inside the last box;
//   MMA     (one warp): S_w = Q_w K^T (both operands in shared memory), O_w += P_w V (P_w from TMEM). While group 0 works on
//           its scores the tensor cores run the other stream's products.
// With heads of 256 elements O takes half of the TMEM: there is one stream, and its scores have two buffers that take turns, so
// that the next tile's are computed while the softmax is at this one's.
// What bounds it: a tile of one stream is 1024 cycles of products (heads of 128), 16384 exponentials (1024 cycles of the
// special-function units, a quarter of them moved to the FMA pipes) and about 900 more of reading, comparing and writing, so two
// streams keep the tensor cores at most busy and the softmax is never far behind. Measured: 2940 cycles for a tile of both streams
// where the products need 2048; a prompt of 8192, 32 heads over 4 of 128, bf16: 439 to 452 us, 1.22 PFLOP/s (73 % of the measured
// burst rate), and 521 to 531 us in long runs, where the power cap lowers the clock.
// The maximum that scales a row's sums is only moved when the row's maximum has grown by more than 2^8 (the probabilities then
// reach 2^8 at most, far inside fp16 and fp32), so rescaling O_w, a round trip through the registers, is rare.
// The values of positions past the sequence's end inside the last box may be anything, and 0 x NaN is NaN: the keys' warp zeroes
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
  static constexpr int STAGES = HD == 64 ? 8 : 4;
  static constexpr uint32_t OUT = 4096;                      // a softmax warp's buffer for 32 rows on their way out, 128 bytes each
  static constexpr int N_BARS = 3 * STAGES + 3 * STREAMS + 8 + 2 * 4 + 1;
  static constexpr uint32_t SMEM = 1024 + STREAMS * Q_TILE + STAGES * STAGE + 4 * STREAMS * OUT + 8 * N_BARS + 16;
  static constexpr uint32_t S_COL = 0, O_COL = 256;          // S_w at 128 w (P_w over its first half), O_w at 256 + HD w
  static_assert(SMEM <= 232448, "shared memory budget");
  static_assert((ATTN_MAX_SEQ + 1) * 8 <= STAGES * STAGE, "the prefix sums fit the ring");
};

CLB_DEV void tma_load_4d(void *dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
               : "memory");
}

CLB_DEV uint32_t upto(int i) { return i < 0 ? 0u : i >= 31 ? ~0u : (2u << i) - 1u; }   // bits 0 .. i

CLB_DEV void tma_load_3d(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_addr(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
               : "memory");
}

// 2^x for x up to 127, two at a time on the FMA pipes: x = n + f with n the nearest integer (by adding 1.5 * 2^23) and f in
// [-0.5, 0.5]; 2^f by a polynomial of degree 5 with constant term 1, fitted to the least relative error (1.6e-7 in fp32); n
// goes into the exponent. Below -127, -infinity included, the result is exactly 0 (n = -127, f = 0).
CLB_DEV float2 exp2_poly(float2 x) {
  x = make_float2(fmaxf(x.x, -127.f), fmaxf(x.y, -127.f));
  const float2 magic = make_float2(12582912.f, 12582912.f);
  const float2 t = fadd2(x, magic), f = fsub2(x, fsub2(t, magic));
  float2 p = make_float2(0.0013264707522466779f, 0.0013264707522466779f);
  p = ffma2(p, f, make_float2(0.00967151764780283f, 0.00967151764780283f));
  p = ffma2(p, f, make_float2(0.05550733953714371f, 0.05550733953714371f));
  p = ffma2(p, f, make_float2(0.24022242426872253f, 0.24022242426872253f));
  p = ffma2(p, f, make_float2(0.6931470036506653f, 0.6931470036506653f));
  p = ffma2(p, f, make_float2(1.f, 1.f));
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}

// What the roles need to know of an item; n 0: the run has ended.
struct __align__(16) TcItem {
  int n, i0, sinks, start;     // this CTA's tiles [i0, i0 + n) of the item; tile i is i below sinks, else start + i
  int s, head, kv, row;        // sequence, key/value head, length, first token's row
  int tokens, lo, hi, whole;   // tokens, positions of the first and last, whether all of its tiles are here
  int pieces, pad[3];          // CTAs that hold the rest of an item that begins here
  CLB_DEV int tile(int i) const { return i0 + i + (i0 + i < sinks ? 0 : start); }
};
constexpr int ITEMS = 4;       // items in shared memory at once

template <typename C, typename O, int HD>
__global__ void __launch_bounds__(TcAttn<HD>::THREADS, 1)
    attn_tc_kernel(const AttnArgs g, const int box, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v) {
  using S = TcAttn<HD>;
  constexpr int N = S::N, ST = S::STREAMS;
  constexpr bool BF16 = __is_same(C, __nv_bfloat16);
  extern __shared__ uint8_t raw[];
  __shared__ TcItem items[ITEMS];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t *ring = sm + ST * S::Q_TILE;
  uint8_t *out_sm = ring + S::STAGES * S::STAGE;
  uint64_t *kv_full = reinterpret_cast<uint64_t *>(out_sm + 4 * ST * S::OUT), *kv_free = kv_full + S::STAGES;
  uint64_t *q_full = kv_free + S::STAGES, *q_free = q_full + ST, *s_full = q_free + ST, *p_half = s_full + 2, *o_full = p_half + 4, *pv_done = o_full + ST;
  uint64_t *item_full = pv_done + 2, *item_free = item_full + ITEMS, *v_whole = item_free + ITEMS, *mma_done = v_whole + S::STAGES;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mma_done + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
  const clb200_attn &a = g.a;
  const int tps = 128 / g.group;   // new tokens per stream

  int64_t *prefix = reinterpret_cast<int64_t *>(ring);
  attn_prefix<N>(g, prefix, cta);
  AttnRun<N> run;
  if (warp == 4 * ST + 2) run.init(g, prefix, cta);
  if (tid == 0) {
    g.joins[cta] = make_int4(0, 0, 0, 0);
    for (int i = 0; i < S::STAGES; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_free[i], 1); mbar_init(&v_whole[i], 1); }
    for (int w = 0; w < ST; ++w) {
      mbar_init(&q_full[w], 1);
      mbar_init(&q_free[w], 1);
      mbar_init(&o_full[w], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&pv_done[w], 1);
      mbar_init(&p_half[2 * w], 4);
      mbar_init(&p_half[2 * w + 1], 4);
    }
    for (int i = 0; i < ITEMS; ++i) { mbar_init(&item_full[i], 1); mbar_init(&item_free[i], 4 * ST + 3); }   // warps that read items
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
  uint32_t it = 0;   // items taken
  // The next item, by a whole warp; n 0 at the end of the run, and when the wait runs out (ok false).
  auto next_item = [&](TcItem &x) {
    const uint32_t k = it % ITEMS;
    if (!wait_bar(&item_full[k], (it / ITEMS) & 1)) { ok = false; x.n = 0; return; }
    x = items[k];
    ++it;
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_free[k]);
  };

  if (warp >= 4 * ST) {
    if constexpr (ST == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 4 * ST + 2) {   // ---- items
      for (;; ++it) {
        const uint32_t k = it % ITEMS;
        if (it >= ITEMS && !wait_bar(&item_free[k], (it / ITEMS - 1) & 1)) { ok = false; break; }
        TcItem x{};
        while (run.more() && x.n == 0) {
          const AttnSpan p = attn_span<N>(g, run.q, run.qt);
          x.n = run.tiles(g, p);
          x.i0 = run.first(g); x.sinks = p.sinks; x.start = p.start;
          x.s = run.s; x.head = run.head; x.kv = run.q.kv; x.row = run.q.row + run.qt * g.tpi;
          x.tokens = min(g.tpi, run.q.nq - run.qt * g.tpi); x.lo = p.lo; x.hi = p.hi; x.whole = x.n == p.nt;
          x.pieces = x.i0 == 0 && !x.whole ? run.pieces(p.nt - x.n) : 0;
          run.advance(g, p);
        }
        if (lane == 0) {
          items[k] = x;
          mbar_arrive(&item_full[k]);
        }
        if (x.n == 0) break;
      }
    } else if (warp == 4 * ST + 3) {   // ---- queries
      TcItem x;
      uint32_t q_cnt[2] = {0, 0};
      for (next_item(x); ok && x.n; next_item(x)) {
#pragma unroll
        for (int w = 0; w < ST; ++w) {
          if (x.tokens <= w * tps) continue;
          if (q_cnt[w] && !wait_bar(&q_free[w], (q_cnt[w] - 1) & 1)) { ok = false; break; }
          ++q_cnt[w];
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[w], static_cast<uint32_t>(tps * g.group) * HD * 2);
#pragma unroll
            for (int cb = 0; cb < HD / 64; ++cb) tma_load_3d(sm + w * S::Q_TILE + cb * (128 * 128), &map_q, 64 * cb, x.head * g.group, x.row + w * tps, &q_full[w]);
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int w = 0; w < ST; ++w)   // every copy issued has landed before the CTA exits
        if (q_cnt[w] && !wait_bar(&q_full[w], (q_cnt[w] - 1) & 1)) ok = false;
    } else if (warp == 4 * ST) {   // ---- keys and values
      uint32_t cnt = 0;
      const int boxes = N / box;
      const AttnSlot outside{g.kv.n_pages, 0};   // a page past the tensor: zeros
      TcItem x{};
      auto where = [&](int tile) {   // this lane's box of a tile
        const int pos = tile * N + lane * box;
        if (lane >= boxes || pos >= x.kv || attn_hidden(g, x.lo, pos, box)) return outside;
        const AttnSlot at = attn_slot(g, x.s, pos);
        return at.page < 0 ? outside : at;
      };
      auto load = [&](const CUtensorMap &map, const AttnSlot &at) -> bool {
        const uint32_t st = cnt % S::STAGES;
        if (cnt >= S::STAGES && !wait_bar(&kv_free[st], (cnt / S::STAGES - 1) & 1)) return false;
        if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], S::STAGE);
        __syncwarp();
        if (lane < boxes) {
          uint8_t *dst = ring + st * S::STAGE + lane * box * 128;
#pragma unroll
          for (int cb = 0; cb < HD / 64; ++cb) tma_load_4d(dst + cb * N * 128, &map, 64 * cb, x.head, at.slot, at.page, &kv_full[st]);
        }
        ++cnt;
        return true;
      };
      for (next_item(x); ok && x.n; next_item(x)) {   // in the order the products take them; pages are looked up two tiles ahead
        AttnSlot at = where(x.tile(0)), next = x.n > 1 ? where(x.tile(1)) : outside;
        ok = load(map_k, at);
        for (int j = 0; ok && j < x.n; ++j) {
          const AttnSlot ahead = j + 2 < x.n ? where(x.tile(j + 2)) : outside;
          if (j + 1 < x.n) ok = load(map_k, next);
          if (ok) ok = load(map_v, at);
          at = next;
          next = ahead;
        }
        const int left = x.kv - x.tile(x.n - 1) * N;
        if (ok && left < N) {   // values past the sequence's end in the item's last tile: zeros, since 0 x NaN is NaN
          const uint32_t vs = (cnt - 1) % S::STAGES;
          if (!wait_bar(&kv_full[vs], ((cnt - 1) / S::STAGES) & 1)) { ok = false; break; }
          for (int i = lane; i < (N - max(left, 0)) * 8 * (HD / 64); i += 32) {
            const int c = i & 7, cb = (i >> 3) % (HD / 64), row = max(left, 0) + (i >> 3) / (HD / 64);
            *reinterpret_cast<uint4 *>(ring + vs * S::STAGE + cb * N * 128 + row * 128 + 16 * c) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_whole[vs]);
        }
        if (!ok) break;
      }
      // every copy issued has landed before the CTA exits (already so unless a wait gave up)
      for (uint32_t v = cnt > S::STAGES ? cnt - S::STAGES : 0; v < cnt; ++v)
        if (!wait_bar(&kv_full[v % S::STAGES], (v / S::STAGES) & 1)) ok = false;
    } else if (tc::elect_one()) {   // ---- MMA: one thread, whose every instruction is on the path of both streams
      constexpr uint32_t ID_S = tc::idesc_half(BF16, false, 128, N), ID_O = tc::idesc_half(BF16, true, 128, HD);
      const uint32_t q_lo = tc::sw128_lo(smem_addr(sm)), k_lo = tc::sw128_lo(smem_addr(ring)), v_lo = tc::sw128_lo(smem_addr(ring), N * 128);
      uint32_t st = 0, round = 0, q_cnt[2] = {0, 0}, p_cnt[2] = {0, 0};   // the next stage and its phase; items and tiles consumed
      uint32_t tails = 0;                                                   // the phase of each stage's v_whole
      auto scores = [&](int w, int b, uint32_t k) {   // S_b = Q_w K^T
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          tc::mma_ss(tmem + S::S_COL + 128 * b, q_lo + w * (S::Q_TILE / 16) + (kk / 4) * (128 * 128 / 16) + 2 * (kk % 4), k + (kk / 4) * (N * 128 / 16) + 2 * (kk % 4), ID_S, kk != 0);
        tc::commit(&s_full[b]);
      };
      auto stage = [&]() {   // the next stage, once it is full
        const uint32_t k = st;
        if (!wait_bar(&kv_full[k], round)) ok = false;
        if (++st == S::STAGES) { st = 0; round ^= 1; }
        return k;
      };
      for (;; ++it) {
        const uint32_t slot = it % ITEMS;
        if (!wait_bar(&item_full[slot], (it / ITEMS) & 1)) { ok = false; break; }
        const int n = items[slot].n;
        const bool two = ST == 2 && items[slot].tokens > tps;                                  // whether the second stream has rows
        const bool tail = n > 0 && items[slot].kv - items[slot].tile(n - 1) * N < N;           // whether the last values are mended
        mbar_arrive(&item_free[slot]);
        if (n == 0) break;
        uint32_t ks = stage(), vs;
#pragma unroll
        for (int w = 0; w < ST; ++w) {
          if (w == 1 && !two) break;
          if (!wait_bar(&q_full[w], q_cnt[w]++ & 1)) ok = false;
          if (!ok) break;
          scores(w, ST == 1 ? p_cnt[0] & 1 : w, k_lo + ks * (S::STAGE / 16));
          if (n == 1) tc::commit(&q_free[w]);
        }
        if (!ok) break;
        tc::commit(&kv_free[ks]);
        for (int j = 0; j < n; ++j) {
          const bool more = j + 1 < n;
          if (more) ks = stage();
          if constexpr (ST == 1) {   // the next tile's scores, in the other buffer, while the softmax is at this one's
            if (more && ok) {
              scores(0, (p_cnt[0] + 1) & 1, k_lo + ks * (S::STAGE / 16));
              tc::commit(&kv_free[ks]);
              if (j + 2 == n) tc::commit(&q_free[0]);
            }
          }
          vs = stage();
          if (tail && !more) {
            if (!wait_bar(&v_whole[vs], (tails >> vs) & 1)) ok = false;
            tails ^= 1u << vs;
          }
          if (!ok) break;
          const uint32_t v = v_lo + vs * (S::STAGE / 16), k = k_lo + ks * (S::STAGE / 16);
#pragma unroll
          for (int w = 0; w < ST; ++w) {
            if (w == 1 && !two) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // (one stream: the buffers take turns, each with its own barriers and every other tile)
              const int b = ST == 1 ? p_cnt[0] & 1 : w;
              if (!wait_bar(&p_half[2 * b + h], (ST == 1 ? p_cnt[0] >> 1 : p_cnt[w]) & 1)) ok = false;
              if (!ok) break;
              tc::fence_after_sync();
#pragma unroll
              for (int kk = 0; kk < N / 32; ++kk)
                tc::mma_ts(tmem + S::O_COL + HD * w, tmem + S::S_COL + 128 * b + 8 * (N / 32 * h + kk), v + 128 * (N / 32 * h + kk), ID_O,
                           (h != 0 || kk != 0) ? true : j != 0);
            }
            ++p_cnt[w];
            if (!ok) break;
            if constexpr (ST == 1) {
              tc::commit(&pv_done[(p_cnt[0] - 1) & 1]);
              if (!more) tc::commit(&o_full[0]);
            } else {
              if (more) scores(w, w, k);
              else tc::commit(&o_full[w]);
              if (j + 2 == n) tc::commit(&q_free[w]);
            }
          }
          if (!ok) break;
          tc::commit(&kv_free[vs]);
          if (ST == 2 && more) tc::commit(&kv_free[ks]);
        }
        if (!ok) break;
      }
      tc::commit(mma_done);   // the TMEM is released only after every MMA issued has completed
      if (!wait_bar(mma_done, 0)) ok = false;
    }
  } else {   // ---- softmax group w, a row per thread
    if constexpr (ST == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int w = warp >> 2, r = tid & 127, tr = attn_token(g, r);
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_col0 = tmem + lanes + S::S_COL + 128 * w, o_col = tmem + lanes + S::O_COL + HD * w;
    const float sc = a.scale * LOG2E;
    uint32_t o_cnt = 0, s_cnt = 0;
    TcItem x_;
    for (next_item(x_); ok && x_.n; next_item(x_)) {
      const TcItem x = x_;
      if (x.tokens <= w * tps) continue;
      const int pos = x.lo + w * tps + tr;
      const bool row_live = r < tps * g.group && w * tps + tr < x.tokens;
      float m = -INFINITY;
      float2 l0 = make_float2(0.f, 0.f), l1 = l0;
      for (int j = 0; j < x.n; ++j) {
        const int b = ST == 1 ? s_cnt & 1 : w;   // the buffer
        const uint32_t s_col = ST == 1 ? s_col0 + 128 * b : s_col0;
        if (!wait_bar(&s_full[b], (ST == 1 ? s_cnt >> 1 : s_cnt) & 1)) { ok = false; break; }
        ++s_cnt;
        tc::fence_after_sync();
        uint32_t xr[N];
        float *v = reinterpret_cast<float *>(xr);
#pragma unroll
        for (int c = 0; c < N / 32; ++c) tc::ld_x32_async(s_col + 32 * c, xr + 32 * c);
#pragma unroll
        for (int c = 0; c < N / 32; ++c) tc::wait_ld_x32(xr + 32 * c);
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < N; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], v[i], v[i + 1]);
        const int p0 = x.tile(j) * N;
        // some row of the stream does not see the whole tile
        if (p0 + N - 1 > x.lo + w * tps || (a.window > 0 && p0 <= x.hi - a.window && p0 + N - 1 >= a.sinks)) {
          const int hi = pos - p0, lo = a.window > 0 ? pos - a.window - p0 : -1, sk = a.window > 0 ? a.sinks - p0 : 0;
          mx[0] = mx[1] = mx[2] = mx[3] = -INFINITY;
#pragma unroll
          for (int c = 0; c < N / 32; ++c) {
            const uint32_t seen = upto(hi - 32 * c) & ~(upto(lo - 32 * c) & ~upto(sk - 1 - 32 * c));
#pragma unroll
            for (int i = 0; i < 32; ++i) v[32 * c + i] = seen & (1u << i) ? v[32 * c + i] : -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], v[32 * c + i], v[32 * c + i + 1]);
          }
        }
        const float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
        // also where m is still -infinity; rows that are nobody's hold anything and have no say, so that the bits do not hang on them
        if (__any_sync(FULL_MASK, row_live && mn > m + 8.0f)) {
          const float mb = fmaxf(m, mn), f = m == -INFINITY ? 0.f : exp2_approx(m - mb);
          m = mb;
          l0.x *= f; l0.y *= f; l1.x *= f; l1.y *= f;
          if (j > 0) {   // O_w is at rest once the products before this tile are complete: they came before its scores, or are waited for
            // one stream: tile s_cnt - 2's products, on the barrier of its buffer (the tile before it there was done long before
            // this tile's scores: a parity tells one phase from the next only)
            if (ST == 1 && !wait_bar(&pv_done[s_cnt & 1], ((s_cnt - 2) >> 1) & 1)) { ok = false; break; }
            if (ST == 1) tc::fence_after_sync();
#pragma unroll 1
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
        for (int h = 0; h < 2; ++h) {   // in halves: the product starts on the first while the second is computed
          uint32_t p[N / 4];
#pragma unroll
          for (int i = 0; i < N / 4; ++i) {
            float2 e = ffma2(make_float2(v[N / 2 * h + 2 * i], v[N / 2 * h + 2 * i + 1]), sc2, nz);
            if (i % 4 == 3) {   // one pair in four on the FMA pipes: the special-function unit alone would be the limit
              e = exp2_poly(e);
            } else {
              e.x = exp2_approx(e.x);
              e.y = exp2_approx(e.y);
            }
            if (i & 1) l1 = fadd2(l1, e);
            else l0 = fadd2(l0, e);
            p[i] = pack2<C>(e.x, e.y);
          }
          if constexpr (N == 128) tc::st_x32(s_col + 32 * h, p);
          else tc::st_x16(s_col + 16 * h, reinterpret_cast<const uint32_t(&)[16]>(p));
          tc::wait_st();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_half[2 * b + h]);
        }
      }
      if (!ok) break;
      if (x.pieces && tid == 0) g.joins[cta] = make_int4(x.row, x.tokens, x.head, x.pieces);
      if (!wait_bar(&o_full[w], o_cnt++ & 1)) { ok = false; break; }
      tc::fence_after_sync();
      const float l = (l0.x + l0.y) + (l1.x + l1.y), inv = x.whole ? (l > 0.f ? 1.0f / l : 0.f) : 1.0f;
      const int64_t piece = static_cast<int64_t>(2 * cta + (x.i0 == 0 ? 1 : 0)) * g.rows + w * tps * g.group;
      if (!x.whole && r < tps * g.group) g.piece_ml[piece + r] = make_float2(m, l);
      // 128 bytes of every row at a time through shared memory, so that eight lanes store a row's and not each lane its own
      uint8_t *buf = out_sm + warp * S::OUT;
      const int k = lane & 7;
      auto pass = [&](const uint32_t (&u)[32], int c, bool to_piece) {   // u: this lane's row; c: the chunk of 128 bytes
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint4 *>(buf + lane * 128 + ((e ^ (lane & 7)) << 4)) = make_uint4(u[4 * e], u[4 * e + 1], u[4 * e + 2], u[4 * e + 3]);
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int row = 4 * e + (lane >> 3), rr = 32 * (warp & 3) + row, tt = attn_token(g, rr), t = w * tps + tt;
          const uint4 q = *reinterpret_cast<const uint4 *>(buf + row * 128 + ((k ^ (row & 7)) << 4));
          if (rr >= tps * g.group || t >= x.tokens) continue;
          uint8_t *dst = to_piece ? reinterpret_cast<uint8_t *>(g.piece_o + (piece + rr) * HD)
                                  : reinterpret_cast<uint8_t *>(static_cast<O *>(a.out) + (x.row + t) * a.out_stride + (x.head * g.group + rr - tt * g.group) * HD);
          reinterpret_cast<uint4 *>(dst + 128 * c)[k] = q;
        }
        __syncwarp();
      };
      if (x.whole && sizeof(O) == 2) {
#pragma unroll 1
        for (int c = 0; c < HD / 64; ++c) {
          uint32_t o[64], u[32];
          tc::ld_x32_async(o_col + 64 * c, o);
          tc::ld_x32_async(o_col + 64 * c + 32, o + 32);
          tc::wait_ld_x32(o);
          tc::wait_ld_x32(o + 32);
#pragma unroll
          for (int i = 0; i < 32; ++i) u[i] = pack2<O>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
          pass(u, c, false);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tc::ld_x32_async(o_col + 32 * c, o);
          tc::wait_ld_x32(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
          pass(o, c, !x.whole);
        }
      }
      tc::fence_before_sync();
    }
    grid_launch_dependents();
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

// The queries as a tensor (element, head, row): boxes of 64 elements of a group's heads by the tokens of a stream.
bool encode_queries(CUtensorMap *m, const AttnArgs &g) {
  const EncodeTiled fn = encoder();
  if (!fn) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(g.kv.head_dim), static_cast<cuuint64_t>(g.a.n_head), static_cast<cuuint64_t>(g.a.T)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(g.kv.head_dim) * 2, static_cast<cuuint64_t>(g.a.q_stride) * 2};
  const cuuint32_t boxes[3] = {64, static_cast<cuuint32_t>(g.group), static_cast<cuuint32_t>(128 / g.group)}, estr[3] = {1, 1, 1};
  return fn(m, g.kv.type == T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(g.a.q), dims, strides, boxes,
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
  CUtensorMap mq, mk, mv;
  if (!encode_queries(&mq, g) || !encode_pages(&mk, g.kv, g.kv.k, box) || !encode_pages(&mv, g.kv, g.kv.v, box)) return cudaErrorInvalidValue;
  attn_tc_kernel<C, O, HD><<<g.nc, S::THREADS, S::SMEM, st>>>(g, box, mq, mk, mv);
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
