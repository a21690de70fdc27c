// The attention's division of work, shared by its kernels (attn.cu, attn_tc.cu).
//
// An item is one sequence, one key/value head and up to `tpi` of the sequence's new tokens, whose tpi x group rows (row = token
// x group + query head of the group) share every key and value they read. Its keys come in tiles of N positions: those up to
// the last token's position, without the tiles that a window hides from all of its tokens. Every item has at least one tile (a
// fully hidden one gives zeros). The tiles of all items, item after item, each item with `lead` units more at its front for what
// beginning and ending it costs, are dealt to the CTAs in equal runs, so ragged batches and long caches balance by themselves
// (the prompt of 8192: 439 us with a lead of 2, 531 without, when the CTA that got the 40 shortest items took a quarter longer
// than the others); an item that falls into several runs leaves one partial state (running
// maximum, sum, unnormalised values per row) per run in the workspace, and a second kernel joins them. A CTA's run holds at
// most two such pieces: the first item's, when an earlier CTA began it (slot 0), and the last item's, when this CTA begins and
// does not finish it (slot 1).
#pragma once
#include "serve.cuh"

namespace clb {

constexpr int ATTN_MAX_SEQ = 512;   // sequences a launch takes (the host launches once per so many)

struct AttnArgs {
  clb200_kv kv;
  clb200_attn a;
  int *err;
  int group, tpi;     // query heads per key/value head, new tokens per item
  uint32_t group_inv; // (65536 + group - 1) / group: row / group = row * group_inv >> 16 for rows below 4096
  int page_shift;     // log2 of the page size where it is a power of two, else -1
  int nc, min_run;    // CTAs, units a CTA takes at least
  int lead;           // units of an item besides its tiles
  int rows;           // rows of a piece (>= tpi x group)
  float *piece_o;     // [nc][2][rows][head_dim]
  float2 *piece_ml;   // [nc][2][rows] maximum (times log2 e) and sum
  int4 *joins;        // [nc] the item that begins in this CTA and does not end there: its first row, tokens, head, and the
                      // pieces that follow (0: there is no such item)
};

struct AttnSeq {
  int row, nq, kv;   // first row, new tokens (0: nothing to do), length
};
// What the device arrays say of sequence s, made safe: a sequence whose rows or length do not fit is skipped, and reported
// when `report` is set.
CLB_DEV AttnSeq attn_seq(const AttnArgs &g, int s, bool report) {
  const int a = g.kv.q_start[s], z = g.kv.q_start[s + 1], n = max(g.kv.kv_len[s], 0);
  AttnSeq q{a, z - a, n};
  if (z <= a) return AttnSeq{a, 0, n};
  if (a < 0 || z > g.a.T || q.nq > g.a.max_q) {
    if (report) set_error(g.err, ERR_BAD_ROWS);
    q.nq = 0;
  } else if (n > static_cast<int64_t>(g.kv.table_width) * g.kv.page_size) {
    if (report) set_error(g.err, ERR_BAD_PAGE);
    q.nq = 0;
  }
  return q;
}

// The tiles of an item: tile i of nt is i for i < sinks, else start + i.
struct AttnSpan {
  int lo, hi;        // positions of its first and last token (may be negative: they see nothing)
  int sinks, start, nt;
  CLB_DEV int tile(int i) const { return i < sinks ? i : start + i; }
};
template <int N>
CLB_DEV AttnSpan attn_span(const AttnArgs &g, const AttnSeq &q, int qt) {
  AttnSpan p;
  const int first = q.kv - q.nq, t0 = qt * g.tpi;
  p.lo = first + t0;
  p.hi = first + min(t0 + g.tpi, q.nq) - 1;
  const int end = p.hi < 0 ? 1 : p.hi / N + 1;
  p.sinks = 0;
  p.start = 0;
  p.nt = end;
  if (g.a.window > 0) {
    const int w0 = max(p.lo - g.a.window + 1, 0) / N, ns = g.a.sinks >= w0 * N ? w0 : (g.a.sinks + N - 1) / N;
    if (ns < w0) {
      p.sinks = ns;
      p.start = w0 - ns;
      p.nt = ns + end - w0;
    }
  }
  return p;
}
CLB_DEV int attn_token(const AttnArgs &g, int row) { return static_cast<int>((static_cast<uint32_t>(row) * g.group_inv) >> 16); }

// The page and slot of position pos (>= 0) of sequence s; page -1 (and the error word set) when there is none.
struct AttnSlot {
  int page, slot;
};
CLB_DEV AttnSlot attn_slot(const AttnArgs &g, int s, int pos) {
  const clb200_kv &kv = g.kv;
  const int i = g.page_shift >= 0 ? pos >> g.page_shift : static_cast<int>(static_cast<uint32_t>(pos) / static_cast<uint32_t>(kv.page_size));
  AttnSlot r{-1, pos - i * kv.page_size};
  if (i < kv.table_width) r.page = __ldg(kv.table + static_cast<int64_t>(s) * kv.table_stride + i);
  if (r.page < 0 || r.page >= kv.n_pages) {
    set_error(g.err, ERR_BAD_PAGE);
    r.page = -1;
  }
  return r;
}

// Whether row position p sees position j (j below the sequence's length).
CLB_DEV bool attn_sees(const AttnArgs &g, int p, int j) {
  return j <= p && (g.a.window <= 0 || j > p - g.a.window || j < g.a.sinks);
}

// Whether no row from position lo on sees any of the n positions from j on: their page is not looked up then (a cache with a window
// may have given it back), and they come as zeros.
CLB_DEV bool attn_hidden(const AttnArgs &g, int lo, int j, int n) {
  return g.a.window > 0 && j + n - 1 <= lo - g.a.window && j >= g.a.sinks;
}

// The tiles of the sequences before each sequence (prefix [n_seq + 1], shared memory). Every thread of the CTA calls it; it
// synchronises the CTA.
template <int N>
CLB_DEV void attn_prefix(const AttnArgs &g, int64_t *prefix, int cta) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5, n_seq = g.kv.n_seq;
  for (int k0 = 32 * warp; k0 < n_seq; k0 += 32 * nw) {   // a lane per sequence, so that their look-ups run side by side
    AttnSeq t{0, 0, 0};
    if (k0 + lane < n_seq) t = attn_seq(g, k0 + lane, cta == 0);
    const int nqt = (t.nq + g.tpi - 1) / g.tpi;
    int64_t sum = 0;
    if (nqt <= 4)
      for (int i = 0; i < nqt; ++i) sum += attn_span<N>(g, t, i).nt + g.lead;
    // a sequence of many items by the whole warp
    for (unsigned many = __ballot_sync(FULL_MASK, nqt > 4); many; many &= many - 1) {
      const int l = __ffs(many) - 1, n = __shfl_sync(FULL_MASK, nqt, l);
      const AttnSeq u{__shfl_sync(FULL_MASK, t.row, l), __shfl_sync(FULL_MASK, t.nq, l), __shfl_sync(FULL_MASK, t.kv, l)};
      int64_t part = 0;
      for (int i = lane; i < n; i += 32) part += attn_span<N>(g, u, i).nt + g.lead;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(FULL_MASK, part, o);
      if (lane == l) sum = part;
    }
    if (k0 + lane < n_seq) prefix[k0 + lane + 1] = sum * g.kv.n_kv;
  }
  if (threadIdx.x == 0) prefix[0] = 0;
  __syncthreads();
  if (warp == 0) {   // inclusive prefix sums: a lane's share, then the lanes before it
    const int per = (n_seq + 31) / 32, b = lane * per, e = min(b + per, n_seq);
    int64_t sum = 0;
    for (int k = b; k < e; ++k) sum += prefix[k + 1];
    int64_t before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(FULL_MASK, before, o);
      if (lane >= o) before += v;
    }
    before -= sum;
    for (int k = b; k < e; ++k) {
      before += prefix[k + 1];
      prefix[k + 1] = before;
    }
  }
  __syncthreads();
}

// A CTA's run of tiles, walked by whole warps (every lane holds the same state).
template <int N>
struct AttnRun {
  int64_t at, end;        // units of all items: the next, and the first that is another CTA's
  int64_t run;            // units a CTA takes
  int s, head, qt, u0;    // the next item, and its first unit that is this CTA's
  AttnSeq q;

  CLB_DEV void init(const AttnArgs &g, const int64_t *prefix, int cta) {
    const int lane = threadIdx.x & 31, n_seq = g.kv.n_seq;
    const int64_t total = prefix[n_seq];
    run = max((total + g.nc - 1) / g.nc, static_cast<int64_t>(g.min_run));
    at = min(run * cta, total);
    end = min(at + run, total);
    if (at >= end) return;
    int lo = 0, hi = n_seq - 1;   // the last sequence that begins at or before `at`
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= at) lo = mid;
      else hi = mid - 1;
    }
    s = lo;
    q = attn_seq(g, s, false);
    const int64_t per_head = (prefix[s + 1] - prefix[s]) / g.kv.n_kv;
    int64_t r = at - prefix[s];
    head = static_cast<int>(r / per_head);
    r -= head * per_head;
    for (int base = 0;; base += 32) {   // the q tile, 32 at a time
      const int nt = (base + lane) * static_cast<int64_t>(g.tpi) < q.nq ? attn_span<N>(g, q, base + lane).nt + g.lead : 0;
      int64_t sum = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(FULL_MASK, sum, o);
        if (lane >= o) sum += v;
      }
      const unsigned hit = __ballot_sync(FULL_MASK, sum > r);
      if (hit || base * static_cast<int64_t>(g.tpi) >= q.nq) {
        const int l = hit ? __ffs(hit) - 1 : 0;
        qt = base + l;
        u0 = static_cast<int>(r - __shfl_sync(FULL_MASK, sum - nt, l));
        break;
      }
      r -= __shfl_sync(FULL_MASK, sum, 31);
    }
  }
  CLB_DEV bool more() const { return at < end; }
  // This CTA's tiles of the next item: n (0 where its run ends inside the item's lead) from first() on.
  CLB_DEV int first(const AttnArgs &g) const { return max(u0 - g.lead, 0); }
  CLB_DEV int tiles(const AttnArgs &g, const AttnSpan &p) const {
    const int64_t u1 = min(static_cast<int64_t>(p.nt + g.lead), u0 + end - at);
    return static_cast<int>(u1 > g.lead ? u1 - g.lead : 0) - first(g);
  }
  CLB_DEV void advance(const AttnArgs &g, const AttnSpan &p) {
    at += p.nt + g.lead - u0;
    u0 = 0;
    if (at >= end) return;
    if (++qt * g.tpi < q.nq) return;
    qt = 0;
    if (++head < g.kv.n_kv) return;
    head = 0;
    do {
      q = attn_seq(g, ++s, false);
    } while (q.nq == 0 && s + 1 < g.kv.n_seq);
  }
  // For an item that begins in this CTA's run and leaves `rest` tiles: how many CTAs hold them.
  CLB_DEV int pieces(int rest) const { return static_cast<int>((rest + run - 1) / run); }
};

// Waits for an mbarrier phase, for two seconds at most; false when they ran out.
CLB_DEV bool wait_bar(uint64_t *bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_ns();
  do {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
  } while (global_ns() - t0 < 2000000000ull);
  return false;
}

CLB_DEV void cp_async16(uint32_t dst, const void *src, bool take) {   // 16 bytes, or zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
CLB_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int K>
CLB_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(K) : "memory"); }

CLB_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
CLB_DEV float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.4426950408889634f;

// Host: the tcgen05 kernel of attn_tc.cu on an argument block whose rows, tpi and nc are its own (attn_tc_rows(head_dim) rows).
cudaError_t launch_attn_tc(const AttnArgs &g, cudaStream_t st);
constexpr int attn_tc_rows(int head_dim) { return head_dim == 256 ? 128 : 256; }

// Host: raises a kernel's shared-memory limit once per device.
template <typename F>
cudaError_t allow_smem(F *fn, int bytes, bool (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 64 && done[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done[dev] = true;
  return e;
}

}  // namespace clb
