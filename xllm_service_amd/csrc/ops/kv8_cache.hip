// What goes into a paged cache held in 8 bits (kv8.h): block tables and slots of a
// step's new tokens, and their keys and values.
#include <algorithm>

#include "kv8.h"

namespace xllm {

// ---- block tables and slots ------------------------------------------------------
// A sequence of `old` tokens grows to `now`. Its new pages come off the free list in
// the order of (sequence, page), its new tokens stand in the order of (sequence,
// position); both offsets are sums over the sequences before it. Integers only, a few
// KB: bound by a launch and the chain lengths -> sums -> ids -> stores. So every
// workgroup makes the sums for itself, 256 sequences at a time, instead of waiting for
// another one's, and writes its share of tokens and pages, which it finds by halves.
constexpr int KV8_SEQS = 256;              // sequences of a round, threads

__global__ __launch_bounds__(KV8_SEQS) void kv8_plan_kernel(
    int* __restrict__ tables, const int* __restrict__ seq_lens,
    const int* __restrict__ new_lens, const int* __restrict__ free_blocks,
    long* __restrict__ slots, long* __restrict__ positions,
    int* __restrict__ cu_q, int* __restrict__ used, const int n_seqs,
    const int width, const long table_stride, const int n_free,
    const int n_tokens) {
  __shared__ int tok_at[KV8_SEQS + 1], page_at[KV8_SEQS + 1], had[KV8_SEQS];
  __shared__ int sums[2][KV8_SEQS / 64];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int groups = gridDim.x, me = blockIdx.x;
  int tokens = 0, pages = 0;               // of the rounds before
  for (int base = 0; base < n_seqs; base += KV8_SEQS) {
    const int i = base + tid;
    const int old = i < n_seqs ? max(seq_lens[i], 0) : 0;
    const int now = i < n_seqs ? max(new_lens[i], old) : 0;
    const int first = old / KV8_PAGE + (old % KV8_PAGE != 0);
    int t = now - old, p = now / KV8_PAGE + (now % KV8_PAGE != 0) - first;
    const int mine_t = t, mine_p = p;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int ut = __shfl_up(t, off, 64), up = __shfl_up(p, off, 64);
      if (lane >= off) t += ut, p += up;
    }
    if (lane == 63) sums[0][wid] = t, sums[1][wid] = p;
    __syncthreads();
    for (int w = 0; w < wid; w++) t += sums[0][w], p += sums[1][w];
    tok_at[tid + 1] = tokens + t;
    page_at[tid + 1] = pages + p;
    had[tid] = old;
    if (tid == 0) tok_at[0] = tokens, page_at[0] = pages;
    if (me == 0 && i < n_seqs) cu_q[i] = min(tokens + t - mine_t, n_tokens);
    __syncthreads();
    const int n = min(n_seqs - base, KV8_SEQS);
    // the sequence of this round that entry x of a list of sums is in
    auto find = [&](const int* at, int x) {
      int lo = 0;
#pragma unroll
      for (int step = KV8_SEQS / 2; step > 0; step >>= 1)
        if (lo + step < n && at[lo + step] <= x) lo += step;
      return lo;
    };
    // chunks of 256, every groups-th of them
    auto mine = [&](int from) {
      const int c = from / KV8_SEQS, ahead = (me - c % groups + groups) % groups;
      return (c + ahead) * KV8_SEQS + tid;
    };
    const int t1 = min(tok_at[n], n_tokens);
    for (int x = mine(tok_at[0]); x < t1; x += groups * KV8_SEQS) {
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
    for (int x = mine(page_at[0]); x < p1; x += groups * KV8_SEQS) {
      if (x < page_at[0]) continue;
      const int s = find(page_at, x);
      const int col = had[s] / KV8_PAGE + (had[s] % KV8_PAGE != 0) + x - page_at[s];
      if ((unsigned)col < (unsigned)width)
        tables[(base + s) * table_stride + col] = free_blocks[x];
    }
    tokens = tok_at[KV8_SEQS];
    pages = page_at[KV8_SEQS];
    __syncthreads();
  }
  if (me == 0 && tid == 0) {
    cu_q[n_seqs] = min(tokens, n_tokens);
    *used = pages;
  }
  // rows behind the last token
  for (int x = tokens + me * KV8_SEQS + tid; x < n_tokens; x += groups * KV8_SEQS) {
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
  const int groups = (int)std::min<long>(256, most / KV8_SEQS + 1);
  hipLaunchKernelGGL(kv8_plan_kernel, dim3(groups), dim3(KV8_SEQS), 0, stream,
                     tables, seq_lens, new_lens, free_blocks, slots, positions,
                     cu_q, used, n_seqs, width, table_stride, n_free, n_tokens);
}

// ---- keys and values ---------------------------------------------------------------
// A page's new tokens stand side by side in slot_mapping, but for skipped ones among
// them. The first of them has its page's waves, two for each head, keys and values, which read all of them, make
// the page's scale and write it: no two waves write to one page, no atomics, one pass.
// With the page's first token among them the page begins anew, and what none of them
// writes is zero; else its earlier tokens stay, rounded again if the scale has grown.
template <int D>
__global__ __launch_bounds__(256) void kv8_write_kernel(
    unsigned char* __restrict__ k_cache, unsigned char* __restrict__ v_cache,
    float* __restrict__ kv_scale, const unsigned short* __restrict__ k,
    const unsigned short* __restrict__ v, const long* __restrict__ slots,
    const int n_tokens, const int n_kv, const long k_stride, const long v_stride,
    const long n_slots) {
  constexpr int NP = D / 64;               // 16 B of the page per lane
  const int lane = threadIdx.x & 63;
  const int t0 = blockIdx.x;
  const int unit = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 +
                                                  (threadIdx.x >> 6));
  const int head = unit >> 1, val = unit & 1;
  if (head >= n_kv) return;
  auto page_of = [&](int t) {              // -1: none
    const long s = slots[t];
    return s >= 0 && s < n_slots ? s / KV8_PAGE : -1L;
  };
  const long page = page_of(t0);
  if (page < 0) return;
  for (int end = t0; end > 0; end -= 64) {  // the last token before that has a page
    const int t = end - 64 + lane;
    const long p = t >= 0 ? page_of(t) : -1L;
    const unsigned long long any = __ballot(p >= 0);
    if (any == 0) continue;
    if (__ballot(p == page) >> (63 - __clzll(any)) & 1) return;
    break;
  }
  const long at = page * n_kv + head;
  const float was = kv_scale[2 * at + val];
  // lane o < 16: the last token that is written to offset o, -1: none
  int src = -1;
  for (int base = t0; base < n_tokens; base += 64) {
    const int t = base + lane;
    const long p = t < n_tokens ? page_of(t) : -1L;
    // of tokens with another page, the first
    const unsigned long long out = __ballot(p >= 0 && p != page);
    const int n = out == 0 ? 64 : __ffsll(out) - 1;
    const int off = p == page ? (int)(slots[t] % KV8_PAGE) : -1;
    unsigned long long in = __ballot(p == page && lane < n);
    for (; in != 0; in &= in - 1) {
      const int j = __builtin_amdgcn_readfirstlane(__ffsll(in) - 1);
      if (lane == __builtin_amdgcn_readlane(off, j)) src = base + j;
    }
    if (n < 64) break;
  }
  const unsigned have = (unsigned)__ballot(src >= 0);
  const bool anew = have & 1;
  unsigned char* to = (val ? v_cache : k_cache) + at * (KV8_PAGE * D);
  // this lane's 16 values of the page, NP times
  float x[NP][16];
  uint4 old[NP];
  int tok[NP];                             // keys: token of the values
  float big = 0.0f;
  auto take = [&](float f, float& y) {
    y = f;
    const float a = fabsf(f);
    big = fmaxf(big, a < INFINITY ? a : 0.0f);
  };
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int p = lane + 64 * i;           // 16 B of the page
    old[i] = make_uint4(0, 0, 0, 0);
    if (!anew && have != 0xffff)
      old[i] = *reinterpret_cast<const uint4*>(to + p * 16);
    if (!val) {                            // chunk p / 16 of token p % 16
      tok[i] = __shfl(src, p & 15, 64);
      if (tok[i] >= 0) {
        const unsigned short* from =
            k + tok[i] * k_stride + (long)head * D + (p >> 4) * 16;
        const ushort8_t a = *reinterpret_cast<const ushort8_t*>(from);
        const ushort8_t b = *reinterpret_cast<const ushort8_t*>(from + 8);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          take(bf16_to_f32(a.x[j]), x[i][j]);
          take(bf16_to_f32(b.x[j]), x[i][8 + j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; j++) x[i][j] = 0.0f;
      }
    } else {                               // channel p
#pragma unroll
      for (int o = 0; o < 16; o++) {
        x[i][o] = 0.0f;
        if (have >> o & 1) {               // uniform
          const int t = __builtin_amdgcn_readlane(src, o);
          take(bf16_to_f32(v[t * v_stride + (long)head * D + p]), x[i][o]);
        }
      }
    }
  }
  const int e = kv8_exponent(wave_reduce_max(big));
  const float fit = kv8_power(e);
  const float now = anew ? fit : fmaxf(was, fit);
  const float by = 1.0f / now;             // exact: a power of two
  const float again = was / now;           // below 1 where the scale has grown
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int p = lane + 64 * i;
    const bool fresh = val || tok[i] >= 0;
    unsigned u[4];
    const unsigned w[4] = {old[i].x, old[i].y, old[i].z, old[i].w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const unsigned kept = again == 1.0f ? w[j] : kv8_again(w[j], again);
      const unsigned made =
          fresh ? kv8_pack(x[i][4 * j] * by, x[i][4 * j + 1] * by,
                           x[i][4 * j + 2] * by, x[i][4 * j + 3] * by)
                : 0;
      unsigned mask = fresh ? ~0u : 0;     // bytes that are new
      if (val) {
        mask = 0;
#pragma unroll
        for (int b = 0; b < 4; b++)
          if (have >> (4 * j + b) & 1) mask |= 255u << (8 * b);
      }
      u[j] = (made & mask) | (anew ? 0 : kept & ~mask);
    }
    if (fresh || anew || again != 1.0f)
      *reinterpret_cast<uint4*>(to + p * 16) = make_uint4(u[0], u[1], u[2], u[3]);
  }
  if (lane == 0) kv_scale[2 * at + val] = now;
}

void launch_kv8_write(unsigned char* k_cache, unsigned char* v_cache,
                      float* kv_scale, const unsigned short* k,
                      const unsigned short* v, const long* slots, int n_tokens,
                      int n_kv, int D, long k_stride, long v_stride,
                      long n_slots, hipStream_t stream) {
  if (n_tokens == 0 || n_slots == 0) return;
  const dim3 grid((unsigned)n_tokens, (unsigned)((2 * n_kv + 3) / 4));
  auto go = D == 128 ? kv8_write_kernel<128> : kv8_write_kernel<64>;
  hipLaunchKernelGGL(go, grid, dim3(256), 0, stream, k_cache, v_cache, kv_scale, k,
                     v, slots, n_tokens, n_kv, k_stride, v_stride, n_slots);
}

}  // namespace xllm
