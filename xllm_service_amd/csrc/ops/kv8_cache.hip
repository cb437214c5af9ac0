// What goes into a paged cache held in 8 bits (kv8.h): block tables and slots of a
// step's new tokens, and their keys and values.
#include <algorithm>

#include "paged_rows.h"

namespace xllm {

// ---- block tables and slots ------------------------------------------------------
// A sequence of `old` tokens grows to `now`. Its new pages come off the free list in
// the order of (sequence, page), its new tokens stand in the order of (sequence,
// position); both offsets are sums over the sequences before it. Integers only, a few
// KB: bound by a launch and the chain lengths -> sums -> ids -> stores. So every
// workgroup makes the sums for itself, a sequence to a thread, instead of waiting for
// another one's, and writes its share of tokens and pages, which it finds by halves.
// Us in a captured graph, where a launch takes 3.2: one sequence 3.3, 128 that grow by a
// token 4.1, 600 by 36 k tokens 5.8, 1000 by 39 k 6.0. A call from the host takes 5.5,
// with the memory of its results.
//   Sums of 32 bits hold whatever lengths a caller has: those past KV8_LONGEST, 2^20 pages,
// count as that, no sequence counts for more tokens than there is room for (2^20 at most,
// kv8_bindings.cpp), and sums of rounds stop at that room and at 2^30 - 1 pages.
// SEQS: sequences of a round, threads.
constexpr int KV8_LONGEST = (1 << 24) - 1;
template <int SEQS>
__global__ __launch_bounds__(SEQS) void kv8_plan_kernel(
    int* __restrict__ tables, const int* __restrict__ seq_lens,
    const int* __restrict__ new_lens, const int* __restrict__ free_blocks,
    long* __restrict__ slots, long* __restrict__ positions,
    int* __restrict__ cu_q, int* __restrict__ used, const int n_seqs,
    const int width, const long table_stride, const int n_free,
    const int n_tokens) {
  __shared__ int tok_at[SEQS + 1], page_at[SEQS + 1], had[SEQS];
  __shared__ int sums[2][SEQS / 64];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int groups = gridDim.x, me = blockIdx.x;
  int tokens = 0, pages = 0;               // of the rounds before
  for (int base = 0; base < n_seqs; base += SEQS) {
    const int i = base + tid;
    const int old = i < n_seqs ? min(max(seq_lens[i], 0), KV8_LONGEST) : 0;
    const int now = i < n_seqs ? min(max(new_lens[i], old), KV8_LONGEST) : 0;
    const int first = old / KV8_PAGE + (old % KV8_PAGE != 0);
    const int mine_t = min(now - old, n_tokens);
    int t = pf_scan<true>(mine_t);
    int p = pf_scan<true>(now / KV8_PAGE + (now % KV8_PAGE != 0) - first);
    if (lane == 63) sums[0][wid] = t, sums[1][wid] = p;
    __syncthreads();
    for (int w = 0; w < wid; w++) t += sums[0][w], p += sums[1][w];
    tok_at[tid + 1] = tokens + t;
    page_at[tid + 1] = pages + p;
    had[tid] = old;
    if (tid == 0) tok_at[0] = tokens, page_at[0] = pages;
    if (me == 0 && i < n_seqs) cu_q[i] = min(tokens + t - mine_t, n_tokens);
    __syncthreads();
    const int n = min(n_seqs - base, SEQS);
    // the sequence of this round that entry x of a list of sums is in
    auto find = [&](const int* at, int x) {
      int lo = 0;
#pragma unroll
      for (int step = SEQS / 2; step > 0; step >>= 1)
        if (lo + step < n && at[lo + step] <= x) lo += step;
      return lo;
    };
    // chunks of SEQS, every groups-th of them
    auto mine = [&](int from) {
      const int c = from / SEQS, ahead = (me - c % groups + groups) % groups;
      return (c + ahead) * SEQS + tid;
    };
    const int t1 = min(tok_at[n], n_tokens);
    for (int x = mine(tok_at[0]); x < t1; x += groups * SEQS) {
      if (x < tok_at[0]) continue;
      const int s = find(tok_at, x), pos = had[s] + x - tok_at[s];
      const int col = pos / KV8_PAGE;
      const int held = had[s] / KV8_PAGE + (had[s] % KV8_PAGE != 0);
      int id = -1;
      if ((unsigned)col < (unsigned)width) {
        const int at = page_at[s] + col - held;
        if (col < held) id = tables[(base + s) * table_stride + col];
        else if (at < n_free) id = free_blocks[at];
      }
      slots[x] = id < 0 ? -1L : (long)id * KV8_PAGE + pos % KV8_PAGE;
      positions[x] = pos;
    }
    const int p1 = min(page_at[n], n_free);
    for (int x = mine(page_at[0]); x < p1; x += groups * SEQS) {
      if (x < page_at[0]) continue;
      const int s = find(page_at, x);
      const int col = had[s] / KV8_PAGE + (had[s] % KV8_PAGE != 0) + x - page_at[s];
      if ((unsigned)col < (unsigned)width)
        tables[(base + s) * table_stride + col] = free_blocks[x];
    }
    tokens = min(tok_at[SEQS], n_tokens);
    pages = min(page_at[SEQS], (1 << 30) - 1);
    __syncthreads();
  }
  if (me == 0 && tid == 0) {
    cu_q[n_seqs] = tokens;
    *used = pages;
  }
  // rows behind the last token
  for (int x = tokens + me * SEQS + tid; x < n_tokens; x += groups * SEQS) {
    slots[x] = -1;
    positions[x] = 0;
  }
}

void launch_kv8_plan(int* tables, const int* seq_lens, const int* new_lens,
                     const int* free_blocks, long* slots, long* positions,
                     int* cu_q, int* used, int n_seqs, int width,
                     long table_stride, int n_free, int n_tokens,
                     hipStream_t stream) {
  const long most = std::max<long>(n_tokens, n_seqs);
  // more than one round of 256: 300 sequences 5.7 | 4.9 us, 1000 8.5 | 5.1; 128 4.1 | 4.6
  const int threads = n_seqs <= 256 ? 256 : 1024;
  const int groups = (int)std::min<long>(256, most / threads + 1);
  auto go = threads == 256 ? kv8_plan_kernel<256> : kv8_plan_kernel<1024>;
  hipLaunchKernelGGL(go, dim3(groups), dim3(threads), 0, stream, tables, seq_lens,
                     new_lens, free_blocks, slots, positions, cu_q, used, n_seqs, width,
                     table_stride, n_free, n_tokens);
}

// ---- keys and values ---------------------------------------------------------------
// A page's new tokens stand side by side in slot_mapping, but for skipped ones among
// them: a run. A run has waves of its own, one for each head, keys and values, which
// read all of it, make the page's scale and write the page: no two waves write to one
// page, no atomics, one pass. With the page's first token in the run the page begins
// anew, and what none of its tokens writes is zero; else its earlier tokens stay, rounded
// again if the scale has grown.
//
// A wave looks a window of tokens over and takes the runs that begin there, one after the
// other, the next one's values on the way meanwhile. Long windows cost tokens that are a
// run each (1.2 us a run: a wave alone on its SIMD issues its 350 instructions in that),
// short ones waves that find no run, of which 126 k take 25 us to come and go. Us, windows
// of 1 | 2 | 4 | 8 | 16, 8 heads of 128: 7878 tokens of four prompts 28 | 21 | 15.7 | 11.9 |
// 11.5, 2000 of one 25 | 15.7 | 9.9 | 6.6 | 5.5, 300 4.9 | 4.4 | 4.4 | 4.3 | 4.3; a token each
// of 1000 sequences 14.5 | 15.1 | 14.6 | 17.2 | 25, of 256 5.9 | 6.6 | 8.6 | 13.5 | 23.5, of 128
// 4.4 | 5.3 | 7.7 | 12.5 | 22. One token: 3.7, a launch.
//   7878 tokens are 48 MB: 11.2, 4.3 TB/s, of the 5.0 of a large copy. Before, by a wave to each
// token and conversions of each value by itself, 47.4.
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;

template <int D, bool VAL>
XLLM_DEV void kv8_write_runs(const long* __restrict__ slots, const int n_tokens,
                             const int n_kv, const int head, const int window,
                             const unsigned n_blocks,
                             const unsigned short* __restrict__ rows,
                             const long stride, float* __restrict__ kv_scale,
                             unsigned char* __restrict__ cache) {
  constexpr int NP = D / 64;               // 16 B of the page per lane
  const int lane = threadIdx.x & 63;
  // page * 16 + offset of a token, -1: skipped
  auto slot_at = [&](int t) {
    if (t < 0 || t >= n_tokens) return -1L;
    const long s = slots[t];
    return (unsigned long)s < (unsigned long)n_blocks * KV8_PAGE ? s : -1L;
  };
  // Whether one of FAR tokens from t on has a slot, by loads that are waited for together:
  // padding is long and has none. Us, 64 at a time | so, 8 heads of 128: 10 tokens in front of
  // padding to 8192 rows 33 | 11.4, to 65 k 238 | 45, to 2^20 5630 | 739, but to 256 5.5 | 6.4:
  // less than half as many are looked over 64 at a time.
  constexpr int FAR = 1024;
  auto any_from = [&](int t) {
    long s[FAR / 64];
#pragma unroll
    for (int i = 0; i < FAR / 64; i++)
      s[i] = slots[min(max(t + 64 * i + lane, 0), n_tokens - 1)];
    bool any = false;
#pragma unroll
    for (int i = 0; i < FAR / 64; i++)
      any |= (unsigned long)s[i] < (unsigned long)n_blocks * KV8_PAGE;
    return __any(any);                     // (more than asked for at the ends, if any)
  };
  auto page_of = [](long slot) { return slot < 0 ? -1 : (int)(slot / KV8_PAGE); };
  // lane i has token base + i: the window, one before it, and what follows
  const int base = (int)blockIdx.x * window - 1;
  const long slot = slot_at(base + lane);
  const int page = page_of(slot), off = (int)(slot & (KV8_PAGE - 1));
  typedef unsigned long long mask;
  const mask on = __ballot(page >= 0);
  const mask before = on & ((1ull << lane) - 1);
  const int last = 63 - __clzll(before | 1);
  int prev = __shfl(page, last, 64);
  if (before == 0) prev = -1;
  mask begins = ((2ull << window) - 2) & on;
  if (begins == 0) return;
  if (__builtin_expect(!(on & 1) && base > 0, 0)) {   // only skipped ones: it is further up
    int found = -1;
    for (int end = base; end > 0 && found < 0; end -= 64) {
      if (end > FAR / 2 && !any_from(end - FAR)) {
        end += 64 - FAR;
        continue;
      }
      const int p = page_of(slot_at(end - 64 + lane));
      const mask any = __ballot(p >= 0);
      if (any != 0) found = __builtin_amdgcn_readlane(p, 63 - __clzll(any));
    }
    if (before == 0) prev = found;
  }
  begins &= __ballot(page != prev);
  if (begins == 0) return;

  // where the last of these runs goes on behind the 64 tokens, if it may and many follow
  int next = base + 64;
  if (__builtin_expect(
          n_tokens - next > FAR / 2 &&
              __builtin_amdgcn_readlane(page, 63 - __clzll(on)) ==
                  __builtin_amdgcn_readlane(page, 63 - __clzll(begins)), 0))
    while (next < n_tokens && !any_from(next)) next += FAR;

  struct Run {                             // on its way
    unsigned raw[8 * NP];                  // this lane's new values, in bf16: keys, 16
                                           // channels of a token; values, NP
                                           // neighbouring channels of 16 tokens
    uint4 old[NP];                         // 16 B of the page as it was
    bool fresh[NP];                        // keys: these are new
    long at;                               // page and head
    float was;                             // scale
    unsigned have;                         // offsets with a new token
    int from, n;                           // first token, tokens
  };
  auto place_of = [&](int i) { return 16 * (VAL ? NP * lane + i : lane + 64 * i); };
  auto load = [&](Run& r) {                // the next one
    const int j = __builtin_amdgcn_readfirstlane(__ffsll(begins) - 1);
    begins &= begins - 1;
    const int id = __builtin_amdgcn_readlane(page, j);
    r.at = (long)id * n_kv + head;
    r.was = kv_scale[2 * r.at + VAL];
    // its page's tokens up to the next one of another page
    const mask up = ~0ull << j;
    const mask other = __ballot(page >= 0 && page != id) & up;
    const int end = other == 0 ? 64 : __builtin_amdgcn_readfirstlane(__ffsll(other) - 1);
    const mask in = __ballot(page == id) & up & (end == 64 ? ~0ull : (1ull << end) - 1);
    int src = -1;                          // lane o < 16: offset o's last token
    r.from = base + j;
    const int off0 = __builtin_amdgcn_readlane(off, j);
    r.n = __popcll(in);
    if (__builtin_expect(end < 64 && in == ((1ull << r.n) - 1) << j &&
                             (__ballot(off == off0 + lane - j) & in) == in, 1)) {
      // tokens one after the other
      if (lane >= off0 && lane < off0 + r.n) src = base + j + lane - off0;
    } else {
      mask m = in;                         // of the 64 tokens from b on
      int o = off, b = base;
      for (bool last = end < 64;;) {
        for (; m != 0; m &= m - 1) {
          const int i = __builtin_amdgcn_readfirstlane(__ffsll(m) - 1);
          const int at = __builtin_amdgcn_readlane(o, i);
          if (lane == at) src = b + i;
        }
        if (last) break;
        b = max(b + 64, next);
        if (b >= n_tokens) break;
        const long s = slot_at(b + lane);
        const int p = page_of(s);
        const mask out = __ballot(p >= 0 && p != id);
        m = __ballot(p == id);
        o = (int)(s & (KV8_PAGE - 1));
        if (out != 0) {
          m &= (out & -out) - 1;
          last = true;
        }
        r.n += __popcll(m);
      }
    }
    r.have = (unsigned)__ballot(src >= 0);
    const unsigned char* to = cache + r.at * (KV8_PAGE * D);
#pragma unroll
    for (int i = 0; i < NP; i++) {
      r.old[i] = make_uint4(0, 0, 0, 0);
      if (!(r.have & 1)) r.old[i] = *reinterpret_cast<const uint4*>(to + place_of(i));
    }
#pragma unroll
    for (int o = 0; o < 8 * NP; o++) r.raw[o] = 0;
    if constexpr (!VAL) {
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const int p = lane + 64 * i;       // chunk p / 16 of token p % 16
        const int t = __shfl(src, p & 15, 64);
        r.fresh[i] = t >= 0;
        if (t >= 0) {
          const uint4* from = reinterpret_cast<const uint4*>(
              rows + t * stride + (long)head * D + (p >> 4) * 16);
          const uint4 a = from[0], b = from[1];
          r.raw[8 * i] = a.x, r.raw[8 * i + 1] = a.y;
          r.raw[8 * i + 2] = a.z, r.raw[8 * i + 3] = a.w;
          r.raw[8 * i + 4] = b.x, r.raw[8 * i + 5] = b.y;
          r.raw[8 * i + 6] = b.z, r.raw[8 * i + 7] = b.w;
        }
      }
    } else {
      const unsigned short* from = rows + (long)head * D + NP * lane;
#pragma unroll
      for (int o = 0; o < 16; o++) {
        if (r.have >> o & 1) {             // uniform
          const long t = __builtin_amdgcn_readlane(src, o);
          if constexpr (NP == 2)
            r.raw[o] = *reinterpret_cast<const unsigned*>(from + t * stride);
          else
            r.raw[o / 2] |= (unsigned)from[t * stride] << (16 * (o & 1));
        }
      }
    }
  };
  auto store = [&](const Run& r) {
    // two values to a word, in the order of the page's bytes
    unsigned x[NP][8];
#pragma unroll
    for (int i = 0; i < NP; i++)
#pragma unroll
      for (int c = 0; c < 8; c++)
        x[i][c] = !VAL || NP == 1
                      ? r.raw[8 * i + c]
                      : __builtin_amdgcn_perm(r.raw[(2 * c + 1) % (8 * NP)],
                                              r.raw[(2 * c) % (8 * NP)],
                                              i ? 0x07060302u : 0x05040100u);
    // sizes of bf16 sort like their bits
    u16x2 two = {0, 0};
#pragma unroll
    for (int i = 0; i < NP; i++)
#pragma unroll
      for (int c = 0; c < 8; c++)
        two = __builtin_elementwise_max(
            two, __builtin_bit_cast(u16x2, x[i][c] & 0x7fff7fffu));
    int big = __builtin_amdgcn_readlane(pf_scan<false>(max(two[0], two[1])), 63);
    // rare, uniform: not all finite, or more tokens than places: those that later ones stand
    // in the place of count for the scale too
    const bool twice = r.n > __popc(r.have);
    if (__builtin_expect(big >= 0x7f80 || twice, 0)) {
      big = 0;
#pragma unroll
      for (int i = 0; i < NP; i++)
#pragma unroll
        for (int c = 0; c < 8; c++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int a = (int)(x[i][c] >> (16 * e)) & 0x7fff;
            big = max(big, a < 0x7f80 ? a : 0);
          }
      mask out = twice ? 0 : 1;
      const int id = page_of(slot_at(r.from));
      for (int b = r.from; b < n_tokens && out == 0; b += 64) {
        const int p = page_of(slot_at(b + lane));
        out = __ballot(p >= 0 && p != id);
        mask m = __ballot(p == id);
        if (out != 0) m &= (out & -out) - 1;
        for (; m != 0; m &= m - 1) {
          const long t = b + __builtin_amdgcn_readfirstlane(__ffsll(m) - 1);
          const unsigned short* row = rows + t * stride + (long)head * D;
          for (int e = lane; e < D; e += 64) {
            const int a = row[e] & 0x7fff;
            big = max(big, a < 0x7f80 ? a : 0);
          }
        }
      }
      big = __builtin_amdgcn_readlane(pf_scan<false>(big), 63);
    }
    const bool anew = r.have & 1;
    const float fit = kv8_power(kv8_exponent(__int_as_float(big << 16)));
    const float now = anew ? fit : fmaxf(r.was, fit);
    const float by = 1.0f / now;           // exact: a power of two
    const float again = r.was / now;       // below 1 where the scale has grown
    const bool keep = __builtin_amdgcn_readfirstlane(again == 1.0f);
    unsigned char* to = cache + r.at * (KV8_PAGE * D);
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const bool fresh = VAL || r.fresh[i];
      unsigned u[4], w[4] = {r.old[i].x, r.old[i].y, r.old[i].z, r.old[i].w};
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const unsigned a = x[i][2 * c], b = x[i][2 * c + 1];
        u[c] = kv8_pack(__uint_as_float(a << 16) * by,
                        __uint_as_float(a & 0xffff0000u) * by,
                        __uint_as_float(b << 16) * by,
                        __uint_as_float(b & 0xffff0000u) * by);
      }
      if (!anew) {                         // uniform
        if (!keep) {
#pragma unroll
          for (int c = 0; c < 4; c++) w[c] = kv8_again(w[c], again);
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
          unsigned fill = fresh ? ~0u : 0; // bytes that are new
          if constexpr (VAL) {
            const unsigned f = r.have >> (4 * c) & 15;
            fill = (f & 1) * 0xffu | (f >> 1 & 1) * 0xff00u |
                   (f >> 2 & 1) * 0xff0000u | (f >> 3) * 0xff000000u;
          }
          u[c] = (u[c] & fill) | (w[c] & ~fill);
        }
      }
      if (fresh || anew || !keep)
        *reinterpret_cast<uint4*>(to + place_of(i)) =
            make_uint4(u[0], u[1], u[2], u[3]);
    }
    if (lane == 0) kv_scale[2 * r.at + VAL] = now;
    // rare, uniform: 448 times this scale is past what fp32 and bf16 hold. What has become
    // more than 240 of it is 240, half a step off at most as any other. (Cut before it is
    // written it kept registers that the rest wants: 7878 tokens 9.8 -> 10.2 us)
    if (__builtin_expect(big > 0x7f70, 0)) {
#pragma unroll 1
      for (int i = 0; i < NP; i++) {
        unsigned* at = reinterpret_cast<unsigned*>(to + place_of(i));
#pragma unroll 1
        for (int c = 0; c < 4; c++) {
          const unsigned y = at[c];
          unsigned far = ((y & 0x7f7f7f7fu) + 0x08080808u) & 0x80808080u & ~kv8_nan(y);
          far = (far >> 7) * 0x7fu;
          at[c] = (y & ~far) | (0x77777777u & far);
        }
      }
    }
  };
  // one is loaded while the one before it is written
  Run a, b;
  load(a);
  for (;;) {
    const bool more = begins != 0;
    if (more) load(b);
    store(a);
    if (!more) break;
    a = b;
  }
}

template <int D>
__global__ __launch_bounds__(256) void kv8_write_kernel(
    const long* __restrict__ slots, const int n_tokens, const int n_kv,
    const int window, const unsigned n_blocks, const unsigned short* __restrict__ k,
    const unsigned short* __restrict__ v, const long k_stride, const long v_stride,
    float* __restrict__ kv_scale, unsigned char* __restrict__ k_cache,
    unsigned char* __restrict__ v_cache) {
  const int unit = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 +
                                                  (threadIdx.x >> 6));
  const int head = unit >> 1;
  if (head >= n_kv) return;
  if (unit & 1)
    kv8_write_runs<D, true>(slots, n_tokens, n_kv, head, window, n_blocks, v, v_stride,
                            kv_scale, v_cache);
  else
    kv8_write_runs<D, false>(slots, n_tokens, n_kv, head, window, n_blocks, k,
                             k_stride, kv_scale, k_cache);
}

void launch_kv8_write(unsigned char* k_cache, unsigned char* v_cache,
                      float* kv_scale, const unsigned short* k,
                      const unsigned short* v, const long* slots, int n_tokens,
                      int n_kv, int D, long k_stride, long v_stride, int n_blocks,
                      hipStream_t stream) {
  if (n_tokens == 0) return;
  // at least 3000 waves, windows of at most eight
  const long waves = 2L * n_kv * n_tokens;
  int window = 1;
  while (window < 8 && 2 * window * 3000L <= waves) window *= 2;
  const dim3 grid((unsigned)((n_tokens + window - 1) / window),
                  (unsigned)((2 * n_kv + 3) / 4));
  auto go = D == 128 ? kv8_write_kernel<128> : kv8_write_kernel<64>;
  hipLaunchKernelGGL(go, grid, dim3(256), 0, stream, slots, n_tokens, n_kv, window,
                     (unsigned)n_blocks, k, v, k_stride, v_stride, kv_scale, k_cache,
                     v_cache);
}

}  // namespace xllm
