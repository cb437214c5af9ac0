// Paged attention of few prompt rows over a cache held in 8 bits (kv8.h), bf16 in and
// out, causal.
//
// As in paged_short.h a workgroup has 32 rows, its four waves walk every fourth tile of
// keys without a barrier, and their results meet in LDS at the end. But a tile is 32 keys
// that go from memory to registers, as for decoded rows (kv8_decode.hip, whose order of
// keys, values and channels this is): nothing passes through LDS, a CU holds two
// workgroups, and pulls half as much for a key.
//
// Scores by e4m3 products (queries as the sum of two e4m3 terms, pages' scales in the
// instruction) need no conversion of keys and took 2% less of long chains, but 0.8 us to
// split the queries: 300 tokens of 32/8 heads 9.1 for 8.2.
#pragma once
#include "paged_rows.h"

namespace xllm {

#define K8S_ROWS 32        // rows per workgroup
#define K8S_WAVES 4
#define K8S_KT 32          // keys per tile

// ONE: there is a single sequence
template <int D, bool ONE>
__global__ __launch_bounds__(K8S_WAVES * 64, 2) void kv8_short_kernel(
    const int* __restrict__ block_tables,    // [num_seqs, max_blocks]
    const int* __restrict__ cu_q,            // [num_seqs+1] query offsets
    const int* __restrict__ seq_lens,        // [num_seqs] total key len
    const int n_seqs, const int G, const int n_kv, const int max_blocks,
    const unsigned char* __restrict__ k_cache, const unsigned short* __restrict__ q,
    const unsigned char* __restrict__ v_cache, const float2* __restrict__ kv_scale,
    unsigned short* __restrict__ out,        // [total_q, n_qheads, D]
    const float scale, const long q_stride, const long out_stride,
    const int n_blocks) {
  constexpr int NW = K8S_WAVES;
  constexpr int NL = D / 32;                 // 16 B a lane of a tile's keys, or values
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int PAGE = PF_BS * D;            // bytes
  __shared__ __attribute__((aligned(16))) f32x4 part[NW * DT * 4 * 64];
  __shared__ float2 ml[NW][K8S_ROWS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, c32 = lane & 31;

  // pages of 32 of the wave's tiles from the tb-th on, two lanes a tile, and their scales;
  // of a single sequence they are asked for before its length is known. What lies past
  // the last page is masked; ids of no page are page 0.
  int tb = 0, ids = 0;
  float2 sizes = {0.0f, 0.0f};
  auto look_up = [&](int seq, int kvh) {
    if (max_blocks <= 0) return;
    const int pg = 2 * (wid + NW * (tb + (lane >> 1))) + (lane & 1);
    const int id = block_tables[(long)seq * max_blocks + min(pg, max_blocks - 1)];
    ids = (unsigned)id < (unsigned)n_blocks ? id : 0;
    sizes = kv_scale[(long)ids * n_kv + kvh];
  };
  const int kvh = blockIdx.x % n_kv;
  if (ONE) look_up(0, kvh);
  PfPlace place;
  if (ONE ? !pf_only<K8S_ROWS>(blockIdx.x / n_kv, INT_MAX / 2, cu_q, seq_lens, G,
                               &place)
          : !pf_locate<K8S_ROWS>(blockIdx.x / n_kv, cu_q, seq_lens, n_seqs, G, lane,
                                 &place))
    return;
  const int q_start = place.q_start, q_len = place.q_len;
  const int room = max_blocks * PF_BS;
  const int ctx = max(place.seq_len, 0) - q_len;
  const int seq_len = min(max(place.seq_len, 0), room);
  const int rows = q_len * G;
  const int row0 = place.lt * K8S_ROWS;
  const int rho = row0 + c32;
  const bool row_ok = rho < rows;
  const int qi = rho / G;
  const int head = kvh * G + rho - qi * G;
  const int limit = row_ok ? min(ctx + qi + 1, room) : 0;   // keys this row sees
  const int wmin = min(ctx + row0 / G + 1, room);           // fewest of a row
  const int kmax = min(ctx + (min(row0 + K8S_ROWS, rows) - 1) / G + 1, room);
  const int n = (max(kmax, 0) + K8S_KT - 1) / K8S_KT;       // tiles
  if (!ONE && wid < n) look_up(place.seq, kvh);

  const PagedScore sc = paged_score<false>(PagedMore{}, scale, 0);
  const float c = sc.c;
  // rows past the last one hold its query: their results go nowhere
  const int qr = min(rho, rows - 1), qq = qr / G;
  const unsigned short* qp = q + (long)(q_start + qq) * q_stride +
                             (long)(kvh * G + qr - qq * G) * D + h * 16;
  bf16x8 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ks++)
    qf[ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * (ks & ~1) + 8 * (ks & 1)) ^
             sc.flip;
  f32x16 o_acc[DT];
#pragma unroll
  for (int i = 0; i < DT; i++) o_acc[i] = mr_zero();
  float m = -INFINITY, l = 0.0f;

  const int last_blk = (seq_len - 1) / PF_BS;
  const bool k_odd = (lane >> 2) & 1;        // the page this lane has keys of
  const int k_off = h * 256 + (4 * (c32 >> 3) + (c32 & 3)) * 16;
  struct Tile {
    uint4 k[NL], v[NL];
    float ks, vs;
  };
  // the wave's i-th tile, if there is one
  auto ask = [&](int i, Tile& x) {
    const int t = wid + NW * i;
    if (t >= n) return;
    if (i - tb == 32) {
      tb += 32;
      look_up(place.seq, kvh);
    }
    const int at = 2 * (i - tb);
    const bool two = 2 * t + 1 <= last_blk;
    auto pick = [&](int v, bool odd) {
      const int a = __builtin_amdgcn_readlane(v, at);
      const int b = __builtin_amdgcn_readlane(v, at + 1);
      return two && odd ? b : a;
    };
    const long kp = (long)pick(ids, k_odd) * n_kv + kvh;
    const long vp = (long)pick(ids, h) * n_kv + kvh;
    const uint4* kf = reinterpret_cast<const uint4*>(k_cache + kp * PAGE + k_off);
    const uint4* vf =
        reinterpret_cast<const uint4*>(v_cache + vp * PAGE + c32 * 16);
#pragma unroll
    for (int j = 0; j < NL; j++) x.k[j] = kf[j * 32];
#pragma unroll
    for (int j = 0; j < NL; j++) x.v[j] = vf[j * 32];
    x.ks = __int_as_float(pick(__float_as_int(sizes.x), k_odd));
    x.vs = __int_as_float(pick(__float_as_int(sizes.y), h));
  };
  auto take = [&](int t, Tile& now) {
    const int k0 = t * K8S_KT;
    f32x16 s = mr_zero();
#pragma unroll
    for (int i = 0; i < NL; i++) {
      s = mr_mma(kv8_wide(now.k[i].x, now.k[i].y, now.ks), qf[2 * i], s);
      s = mr_mma(kv8_wide(now.k[i].z, now.k[i].w, now.ks), qf[2 * i + 1], s);
    }
    unsigned sees = 0;                       // this row's keys of the tile, ...
    unsigned short* nan = nullptr;           // ... and values that are NaNs, by channel
    if (k0 + K8S_KT > wmin) {                // uniform: not all rows see all of it
#pragma unroll
      for (int r = 0; r < 16; r++)
        s[r] = k0 + 16 * h + r < limit ? s[r] : -INFINITY;
      // behind the last key: no value, whatever a page holds there
      const int keys = seq_len - k0 - 16 * h;
      bool any = false;
#pragma unroll
      for (int i = 0; i < NL; i++) {
        now.v[i] = kv8_first(now.v[i], keys);
        any |= (kv8_nan(now.v[i].x) | kv8_nan(now.v[i].y) | kv8_nan(now.v[i].z) |
                kv8_nan(now.v[i].w)) != 0;
      }
      now.vs = keys > 0 ? now.vs : 1.0f;
      if (__any(any)) {                      // 0 times a NaN is one
        nan = reinterpret_cast<unsigned short*>(part + wid * (DT * 4 * 64));
#pragma unroll
        for (int i = 0; i < NL; i++)
          nan[(i * 32 + c32) * 2 + h] = kv8_drop_nan(now.v[i]);
        sees = limit - k0 >= 32 ? ~0u : (1u << max(limit - k0, 0)) - 1u;
      }
    }
    float mt = s[0];                         // weights are 2^(c (s - m))
#pragma unroll
    for (int r = 1; r < 16; r++) mt = fmaxf(mt, s[r]);
    mt = pair_max(mt);
    // scaled only where a maximum has grown by more than 2^8, as in paged_rows.h over such
    // pages: 3 x 61-333 behind 0.5-3 k 19.9 -> 18.8
    if (__any((mt - m) * c > 8.0f)) {
      const float m_new = fmaxf(m, mt);
      const float alpha =
          __builtin_amdgcn_exp2f((m - (m_new == -INFINITY ? 0.f : m_new)) * c);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int j = 0; j < DT; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) o_acc[j][r] *= alpha;
    }
    const float mc = m == -INFINITY ? 0.0f : m * c;
    bf16x8 p[2];
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const float a = __builtin_amdgcn_exp2f(fmaf(s[r], c, -mc));
      const float b = __builtin_amdgcn_exp2f(fmaf(s[r + 1], c, -mc));
      const unsigned u = pack_bf16(a, b);
      l = kv8_add(u, l);
      reinterpret_cast<unsigned*>(&p[r >> 3])[(r & 7) >> 1] = u;
    }
#pragma unroll
    for (int j = 0; j < DT; j++) {
      o_acc[j] = mr_mma(kv8_wide(now.v[j].x, now.v[j].y, now.vs), p[0], o_acc[j]);
      o_acc[j] = mr_mma(kv8_wide(now.v[j].z, now.v[j].w, now.vs), p[1], o_acc[j]);
    }
    if (nan != nullptr) {                    // uniform
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const unsigned* of = reinterpret_cast<const unsigned*>(nan);
#pragma unroll
      for (int j = 0; j < DT; j++)
#pragma unroll
        for (int r = 0; r < 16; r++)
          if (of[j * 32 + 8 * (r >> 2) + 4 * h + (r & 3)] & sees) o_acc[j][r] = NAN;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  };
  Tile tiles[2];
  ask(0, tiles[0]);
  for (int i = 0, t = wid; t < n;) {
#pragma unroll
    for (int b = 0; b < 2; b++) {
      if (t >= n) break;
      ask(i + 1, tiles[b ^ 1]);
      take(t, tiles[b]);
      t += NW;
      i++;
    }
  }

  // ---- the waves' results ------------------------------------------------------
  l = pair_sum(l);
  if (h == 0) ml[wid][c32] = make_float2(m == -INFINITY ? m : m * c, l);
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int r = 0; r < 4; r++)
      part[((wid * DT + dt) * 4 + r) * 64 + lane] =
          f32x4{o_acc[dt][4 * r], o_acc[dt][4 * r + 1], o_acc[dt][4 * r + 2],
                o_acc[dt][4 * r + 3]};
  __syncthreads();
  if (!row_ok) return;
  float top = -INFINITY, sum = 0.0f, f[NW];
#pragma unroll
  for (int w = 0; w < NW; w++) top = fmaxf(top, ml[w][c32].x);
#pragma unroll
  for (int w = 0; w < NW; w++) {
    const float2 z = ml[w][c32];
    // a wave without keys has no part in the row
    f[w] = w < n ? __builtin_amdgcn_exp2f(z.x - (top == -INFINITY ? 0.0f : top)) : 0.0f;
    if (w < n) sum += z.y * f[w];
  }
  const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
  // a wave writes its share of the pieces of all rows
  const long to = (long)(q_start + qi) * out_stride + (long)head * D + 4 * h;
#pragma unroll
  for (int i = 0; i < 4 * DT / NW; i++) {
    const int piece = wid * (4 * DT / NW) + i, dt = piece >> 2, r = piece & 3;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < NW; w++)
      if (w < n) o += part[((w * DT + dt) * 4 + r) * 64 + lane] * f[w];
    paged_put<false>(PagedMore{}, out, to + dt * 32 + 8 * r, o[0] * inv, o[1] * inv,
                     o[2] * inv, o[3] * inv);
  }
}

template <int D>
inline void kv8_short(unsigned short* out, const unsigned short* q,
                      const unsigned char* k_cache, const unsigned char* v_cache,
                      const int* block_tables, const int* cu_q, const int* seq_lens,
                      long tokens, int n_seqs, float scale, int n_qheads, int n_kv,
                      int max_blocks, long q_stride, long out_stride,
                      const Kv8Pages& c8, hipStream_t stream) {
  const int G = n_qheads / n_kv;
  auto go = n_seqs == 1 ? kv8_short_kernel<D, true> : kv8_short_kernel<D, false>;
  hipLaunchKernelGGL(
      go, dim3((unsigned)(paged_rows_tiles<K8S_ROWS>(tokens, n_seqs, G) * n_kv)),
      dim3(K8S_WAVES * 64), 0, stream, block_tables, cu_q, seq_lens, n_seqs, G, n_kv,
      max_blocks, k_cache, q, v_cache, c8.scale, out, scale, q_stride, out_stride,
      c8.blocks);
}

}  // namespace xllm
