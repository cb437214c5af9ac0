// Paged attention of decoded rows over a cache held in 8 bits (kv8.h): bf16 in and out.
//
// For one (sequence, key head) the G query heads (G <= 16) are the columns of
// S^T = K Q^T and of O^T += V^T P^T. What the A operands want of a lane lies side by side in
// the pages, so a tile goes from memory to registers in 16 B a lane and is converted
// there, the scale of its page in the same instruction: no LDS, no transposes, no
// barrier in the loop.
//
// Weights have two bf16 terms (16 bits), the second ones in the columns that the heads
// leave (paged_stream.h). Waves have tiles of their own and meet in LDS at the end;
// long sequences are split over workgroups, the last of which merges (paged_merge.h).
//
// Bound by memory where there is much of it: 128 sequences of 1-2 k keys, 32/8 heads of
// 128, 76 to 82 us by card, 5.3 to 4.9 TB/s (a large copy: 5.0; bf16 pages 144 us); 6 of
// 9-20 k, 28/4 heads, whose 92 MB are longer than the cache before memory 23 (40), and 18.8
// where they are partly in it. One of 776 6.7 to 7.1 (8.1): a launch, a chain of table,
// scales and keys, then of four tiles a wave.
#include "kv8.h"
#include "paged_stream.h"

namespace xllm {

// The waves' results in LDS, [4][2 G][D + 4] with second terms apart and their maxima and
// sums, become the workgroup's: its sequence's, or a part of them, of which the last
// workgroup makes the sequence's.
template <int D, bool SPLIT>
XLLM_DEV void kv8_meet(unsigned short* out, float* ws_o, float* ws_ml, const float* mo,
                       const float (*ml_lds)[16][2], int* flag, int seq, int kvh,
                       int part, int parts, int P, int G, int n_kv, int unit,
                       long out_stride, const PagedMeet& meet) {
  constexpr int NW = 4, DP = D + 4;
  const int tid = threadIdx.x, R = 2 * G;
  __syncthreads();
  const long rows_at = ((long)seq * n_kv + kvh) * G * P;
  const auto unit_o = mr_buffer(ws_o + rows_at * D, parts == 1 ? 0 : G * P * D * 4);
  const auto unit_ml = mr_buffer(ws_ml + rows_at * 2, parts == 1 ? 0 : G * P * 8);
  unsigned short* mine = out + (long)seq * out_stride + (long)kvh * G * D;
  auto put = [&](int row, int at, float L, const float (&a)[4]) {
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;       // no keys: zeros
    paged_put<false>(PagedMore{}, mine, (long)row * D + at, a[0] * inv, a[1] * inv,
                     a[2] * inv, a[3] * inv);
  };
  for (int idx = tid; idx < G * (D / 4); idx += NW * 64) {
    const int row = idx / (D / 4), at = idx % (D / 4) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; w++) M = fmaxf(M, ml_lds[w][row][0]);
    const float Mu = M == -INFINITY ? 0.0f : M;
    float L = 0.0f, a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < NW; w++) {
      const float f = __builtin_amdgcn_exp2f(ml_lds[w][row][0] - Mu);
      L += ml_lds[w][row][1] * f;
      const float* from = mo + (w * R + row) * DP + at;
      const float4 y = *reinterpret_cast<const float4*>(from);
      const float4 z = *reinterpret_cast<const float4*>(from + G * DP);
      a[0] += (y.x + z.x) * f; a[1] += (y.y + z.y) * f;
      a[2] += (y.z + z.z) * f; a[3] += (y.w + z.w) * f;
    }
    if (!SPLIT || parts == 1) {
      put(row, at, L, a);
    } else {
      const int slot = row * P + part;
      if (at == 0) mr_store_far2(unit_ml, slot * 8, make_float2(M, L));
      mr_store_far(unit_o, (slot * D + at) * 4,
                   make_float4(a[0], a[1], a[2], a[3]));
    }
  }
  if (!SPLIT || parts == 1 || !paged_last(meet.count + unit, parts, flag)) return;
  // ---- all parts are there ----------------------------------------------------
  for (int idx = tid; idx < G * (D / 4); idx += NW * 64) {
    const int row = idx / (D / 4), at = idx % (D / 4) * 4;
    float M = -INFINITY, L = 0.0f, a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int slot = row * P;
    paged_add_parts<8>(
        [&](int p) { return mr_load_far2(unit_ml, (slot + p) * 8); },
        [&](int p) { return mr_load_far(unit_o, ((slot + p) * D + at) * 4); },
        parts, M, L, a);
    put(row, at, L, a);
  }
}

// G <= 16 on 32x32x16 products (layouts: mfma_rows.h). A tile is 32 keys, two pages.
//
//   keys     row m of A is key 4 (m >> 3) + (m & 3) of page (m >> 2) & 1: then the 16
//            scores that lane half h holds of a column are those of page h, in order
//   values   lane half h gives page h: its 16 bytes of a channel are the operands
//            of both steps that its 16 weights want
//   channels of a key are summed in the order of its 16 B chunks, h taking every
//            second one, queries likewise
template <int D, bool SPLIT>
__global__ __launch_bounds__(256, 2) void kv8_decode_kernel(
    const int* __restrict__ block_tables,    // [num_seqs, max_blocks]
    const int* __restrict__ seq_lens,        // [num_seqs]
    const int G, const int n_kv, const int max_blocks, const int n_blocks,
    const unsigned char* __restrict__ k_cache,
    const unsigned char* __restrict__ v_cache,
    const float2* __restrict__ kv_scale,     // [blocks, n_kv]: of keys, of values
    const unsigned short* __restrict__ q,    // [num_seqs, n_qheads, D] bf16
    unsigned short* __restrict__ out,        // [num_seqs, n_qheads, D]
    float* __restrict__ ws_o,                // [S*n_qheads][P][D] (P > 1)
    float* __restrict__ ws_ml,               // [S*n_qheads][P][2]
    const float scale, const long q_stride, const long out_stride,
    const PagedSplit split, const PagedMeet meet) {
  constexpr int NW = 4;                      // waves
  constexpr int NL = D / 32;                 // 16 B a lane of a tile's keys, or values
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int PAGE = KV8_PAGE * D;         // bytes
  constexpr int DP = D + 4;                  // rows on other banks
  __shared__ __attribute__((aligned(16))) float mo[NW * 32 * DP];
  __shared__ float ml_lds[NW][16][2];
  __shared__ int flag;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, c32 = lane & 31;
  const int P = SPLIT ? split.parts : 1, units = gridDim.x / P;
  const int part = blockIdx.x / units, unit = blockIdx.x % units;
  const int seq = unit / n_kv, kvh = unit % n_kv;
  const int seq_len = min(seq_lens[seq], max_blocks * KV8_PAGE);
  const int n_tiles = (max(seq_len, 0) + PA_KT - 1) / PA_KT;
  const int parts = SPLIT ? split.of(n_tiles) : 1;
  if (SPLIT && part >= parts) return;
  u64 seen = 0;
  if (SPLIT && parts > 1 && tid == 0) seen = paged_seen(meet.count + unit);
  const int step = parts * NW, i0 = part * NW + wid;

  const int col = c32 & 15;
  const bool second = c32 >= 16;             // second terms of column col
  const unsigned first = second ? 0xffff0000u : 0u;
  const bool row_ok = col < G;
  const int head = kvh * G + (row_ok ? col : 0);
  const PagedScore sc = paged_score<false>(PagedMore{}, scale, 0);
  bf16x8 qf[KS];                             // padding: the first head's query
#pragma unroll
  for (int ks = 0; ks < KS; ks++)
    qf[ks] = *reinterpret_cast<const bf16x8*>(
                 q + (long)seq * q_stride + (long)head * D +
                 16 * ((ks & ~1) + h) + 8 * (ks & 1)) ^
             sc.flip;
  f32x16 o_acc[DT];
#pragma unroll
  for (int i = 0; i < DT; i++) o_acc[i] = mr_zero();
  float m = -INFINITY, l = 0.0f;

  const int* btab = block_tables + (long)seq * max_blocks;
  const int last_blk = (seq_len - 1) / KV8_PAGE;
  // pages of 32 of the wave's tiles from the tb-th on, two lanes a tile, and their
  // scales. What lies past the last page is not used; ids of no page are page 0.
  int tb = 0, ids = 0;
  float2 sizes = {0.0f, 0.0f};
  auto look_up = [&](int n) {
    if (max_blocks <= 0) return;
    const int id = btab[min(2 * (i0 + (n + (lane >> 1)) * step) + (lane & 1),
                            max_blocks - 1)];
    ids = (unsigned)id < (unsigned)n_blocks ? id : 0;
    sizes = kv_scale[(long)ids * n_kv + kvh];
  };
  const bool k_odd = (lane >> 2) & 1;        // the page this lane has keys of
  const int k_off = h * 256 + (4 * (c32 >> 3) + (c32 & 3)) * 16;
  struct Tile {
    uint4 k[NL], v[NL];
    float ks, vs;
  };
  auto load = [&](int n, Tile& x) {
    const int t = i0 + n * step, at = 2 * (n - tb);
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
    for (int i = 0; i < NL; i++) x.k[i] = kf[i * 32];
#pragma unroll
    for (int i = 0; i < NL; i++) x.v[i] = vf[i * 32];
    x.ks = __int_as_float(pick(__float_as_int(sizes.x), k_odd));
    x.vs = __int_as_float(pick(__float_as_int(sizes.y), h));
  };
  look_up(0);
  if (SPLIT && parts > 1 && tid == 0) paged_open(meet.count + unit, seen, meet.tag);
  Tile tiles[2];
  // tile n, if there is one, into its place
  auto ask = [&](int n, Tile& x) {
    if (i0 + n * step >= n_tiles) return;
    if (n - tb == 32) {
      tb += 32;
      look_up(tb);
    }
    load(n, x);
  };
  auto take = [&](int t, Tile& now) {
    f32x16 s[1] = {mr_zero()};
#pragma unroll
    for (int i = 0; i < NL; i++) {
      s[0] = mr_mma(kv8_wide(now.k[i].x, now.k[i].y, now.ks), qf[2 * i], s[0]);
      s[0] = mr_mma(kv8_wide(now.k[i].z, now.k[i].w, now.ks), qf[2 * i + 1], s[0]);
    }
    if (t == n_tiles - 1) {                  // uniform
      // behind the last key: no score, and no value, whatever a page holds there
      const int keys = seq_len - t * PA_KT - 16 * h;
#pragma unroll
      for (int r = 0; r < 16; r++) s[0][r] = r < keys ? s[0][r] : -INFINITY;
#pragma unroll
      for (int i = 0; i < NL; i++) now.v[i] = kv8_first(now.v[i], keys);
    }
    const float c = sc.c;                    // weights are 2^(c (s - m))
    float mt = s[0][0];
#pragma unroll
    for (int r = 1; r < 16; r++) mt = fmaxf(mt, s[0][r]);
    mt = pair_max(mt);
    if (__any(mt > m)) {
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
      float a = __builtin_amdgcn_exp2f(fmaf(s[0][r], c, -mc));
      float b = __builtin_amdgcn_exp2f(fmaf(s[0][r + 1], c, -mc));
      l += a + b;
      a -= __uint_as_float(__float_as_uint(a) & first);
      b -= __uint_as_float(__float_as_uint(b) & first);
      reinterpret_cast<unsigned*>(&p[r >> 3])[(r & 7) >> 1] =
          __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
#pragma unroll
    for (int j = 0; j < DT; j++) {
      o_acc[j] = mr_mma(kv8_wide(now.v[j].x, now.v[j].y, now.vs), p[0], o_acc[j]);
      o_acc[j] = mr_mma(kv8_wide(now.v[j].z, now.v[j].w, now.vs), p[1], o_acc[j]);
    }
  };
  ask(0, tiles[0]);                          // (two ahead: no faster)
  for (int n = 0, t = i0; t < n_tiles;) {
#pragma unroll
    for (int b = 0; b < 2; b++) {
      if (t >= n_tiles) break;
      ask(n + 1, tiles[b ^ 1]);
      take(t, tiles[b]);
      t += step;
      n++;
    }
  }
  l = pair_sum(l);

  // ---- the waves' results meet in LDS ----------------------------------------
  const int R = 2 * G;                                   // second terms apart
  if (row_ok) {
    if (h == 0 && !second) {
      ml_lds[wid][col][0] = m == -INFINITY ? m : m * sc.c;
      ml_lds[wid][col][1] = l;
    }
    float* mine = mo + (wid * R + (second ? G : 0) + col) * DP + 4 * h;
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<float4*>(mine + i * 32 + 2 * r) =
            make_float4(o_acc[i][r], o_acc[i][r + 1], o_acc[i][r + 2],
                        o_acc[i][r + 3]);
  }
  kv8_meet<D, SPLIT>(out, ws_o, ws_ml, mo, ml_lds, &flag, seq, kvh, part, parts, P, G,
                     n_kv, unit, out_stride, meet);
}

// G <= 8 on 16x16x32 products, which have half the columns: half the scores to a lane, 112
// registers for sums, queries and a tile's keys and values where the other kernel has 160,
// and so three waves to a SIMD, four for 64-wide heads. Us, that kernel | this one: 6 x
// 9-20 k of 28/4 heads 26.5 | 23.0, 16 x 0.5-4 k of 32/8 20.2 | 17.6, 24 x 0.6-1.4 k 14.7 | 12.7,
// 1 x 300 6.2 | 5.4, 128 x 300 23.4 | 20.8, 128 x 1-2 k 82.6 | 81.7 (1024 workgroups are two
// full turns of it and one and a third of these), 48 of 12 heads of 64 22.7 | 20.6. A tile
// is 64 keys, four pages, and quarter q of the lanes (l >> 4) has page q:
//
//   keys     row m of set t is token 4 t + (m & 3) of page m >> 2; after four sets a lane
//            holds the 16 scores of its page, in order
//   values   16 bytes of a channel are the operands of both steps
//
// Keys of the next tile are asked for when this one's are multiplied, its values when
// this one's are: into the same registers.
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f4;
XLLM_DEV f4 kv8_mma16(bf16x8 a, bf16x8 b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// largest / sum of the four lanes that share l & 15
XLLM_DEV float kv8_max4(float v) {
  const unsigned u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
XLLM_DEV float kv8_sum4(float v) {
  const unsigned u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

constexpr int KV8_KT = 64;                   // keys of a tile

template <int D, bool SPLIT>
__global__ __launch_bounds__(256, D == 128 ? 3 : 4) void kv8_decode16_kernel(
    const int* __restrict__ block_tables, const int* __restrict__ seq_lens,
    const int G, const int n_kv, const int max_blocks, const int n_blocks,
    const unsigned char* __restrict__ k_cache,
    const unsigned char* __restrict__ v_cache,
    const float2* __restrict__ kv_scale, const unsigned short* __restrict__ q,
    unsigned short* __restrict__ out, float* __restrict__ ws_o,
    float* __restrict__ ws_ml, const float scale, const long q_stride,
    const long out_stride, const PagedSplit split, const PagedMeet meet) {
  constexpr int NW = 4;                      // waves
  constexpr int NC = D / 64;                 // 16 B a lane of a set's keys
  constexpr int DT = D / 16;
  constexpr int PAGE = KV8_PAGE * D;         // bytes
  constexpr int DP = D + 4;                  // rows on other banks
  __shared__ __attribute__((aligned(16))) float mo[NW * 16 * DP];
  __shared__ float ml_lds[NW][16][2];
  __shared__ int flag;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int quad = lane >> 4, c16 = lane & 15;
  const int P = SPLIT ? split.parts : 1, units = gridDim.x / P;
  const int part = blockIdx.x / units, unit = blockIdx.x % units;
  const int seq = unit / n_kv, kvh = unit % n_kv;
  const int seq_len = min(seq_lens[seq], max_blocks * KV8_PAGE);
  const int n_tiles = (max(seq_len, 0) + KV8_KT - 1) / KV8_KT;
  const int parts = SPLIT ? split.of(n_tiles) : 1;
  if (SPLIT && part >= parts) return;
  u64 seen = 0;
  if (SPLIT && parts > 1 && tid == 0) seen = paged_seen(meet.count + unit);
  const int step = parts * NW, i0 = part * NW + wid;

  // pages of 16 of the wave's tiles from the tb-th on, four lanes a tile, and their
  // scales. What lies past the last page is masked; ids of no page are page 0.
  const int* btab = block_tables + (long)seq * max_blocks;
  int tb = 0, ids = 0;
  float2 sizes = {0.0f, 0.0f};
  auto entry = [&](int n) {
    return max_blocks <= 0
        ? 0
        : btab[min(4 * (i0 + (n + (lane >> 2)) * step) + (lane & 3), max_blocks - 1)];
  };
  auto look_up = [&](int id) {
    ids = (unsigned)id < (unsigned)n_blocks ? id : 0;
    sizes = kv_scale[(long)ids * n_kv + kvh];
  };
  const int id0 = entry(0);

  const int col = c16 & 7;
  const bool second = c16 >= 8;              // second terms of column col
  const unsigned first = second ? 0xffff0000u : 0u;
  const bool row_ok = col < G;
  const int head = kvh * G + (row_ok ? col : 0);
  const PagedScore sc = paged_score<false>(PagedMore{}, scale, 0);
  bf16x8 qf[2 * NC];                         // padding: the first head's query
#pragma unroll
  for (int i = 0; i < 2 * NC; i++)
    qf[i] = *reinterpret_cast<const bf16x8*>(
                q + (long)seq * q_stride + (long)head * D +
                16 * (4 * (i >> 1) + quad) + 8 * (i & 1)) ^
            sc.flip;
  __builtin_amdgcn_sched_barrier(0);         // queries are asked for before the wait
  look_up(id0);
  f4 o_acc[DT];
#pragma unroll
  for (int i = 0; i < DT; i++) o_acc[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;

  const int k_page = c16 >> 2;               // of the tile, that this lane has keys of
  const unsigned k_off = quad * 256 + (c16 & 3) * 16, v_off = c16 * 16;
  uint4 kr[4][NC], vr[DT];
  auto load_k = [&](int n) {
    const int at = 4 * (n - tb) + k_page;
    const uint4* from = reinterpret_cast<const uint4*>(
        k_cache + ((long)__shfl(ids, at, 64) * n_kv + kvh) * PAGE + k_off);
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int i = 0; i < NC; i++) kr[t][i] = from[i * 64 + t * 4];
  };
  auto load_v = [&](int n) {
    const int at = 4 * (n - tb) + quad;
    const uint4* from = reinterpret_cast<const uint4*>(
        v_cache + ((long)__shfl(ids, at, 64) * n_kv + kvh) * PAGE + v_off);
#pragma unroll
    for (int i = 0; i < DT; i++) vr[i] = from[i * 16];
  };
  if (SPLIT && parts > 1 && tid == 0) paged_open(meet.count + unit, seen, meet.tag);
  if (i0 < n_tiles) {
    load_k(0);
    load_v(0);
  }
  for (int t = i0, n = 0; t < n_tiles; t += step, n++) {
    const bool more = t + step < n_tiles;
    // (asked for no earlier: the first values would wait for the scales)
    const float ks = __shfl(sizes.x, 4 * (n - tb) + k_page, 64);
    float vs = __shfl(sizes.y, 4 * (n - tb) + quad, 64);
    f4 s[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      s[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < NC; i++) {
        s[j] = kv8_mma16(kv8_wide(kr[j][i].x, kr[j][i].y, ks), qf[2 * i], s[j]);
        s[j] = kv8_mma16(kv8_wide(kr[j][i].z, kr[j][i].w, ks), qf[2 * i + 1], s[j]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) {
      if (n + 1 - tb == 16) {                // this tile's values are on their way
        tb += 16;
        look_up(entry(tb));
      }
      load_k(n + 1);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (t == n_tiles - 1) {                  // uniform
      // behind the last key: no score, and no value, whatever a page holds there
      const int keys = seq_len - t * KV8_KT - KV8_PAGE * quad;
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) s[j][r] = 4 * j + r < keys ? s[j][r] : -INFINITY;
#pragma unroll
      for (int i = 0; i < DT; i++) vr[i] = kv8_first(vr[i], keys);
      vs = keys > 0 ? vs : 1.0f;
    }
    const float c = sc.c;                    // weights are 2^(c (s - m))
    float mt = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
    for (int j = 1; j < 4; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) mt = fmaxf(mt, s[j][r]);
    mt = kv8_max4(mt);
    // Weights of 16 bits and sums round the same whatever they are scaled by: they are
    // scaled anew only where a maximum has grown by more than 2^8.
    if (__any((mt - m) * c > 8.0f)) {
      const float m_new = fmaxf(m, mt);
      const float alpha =
          __builtin_amdgcn_exp2f((m - (m_new == -INFINITY ? 0.f : m_new)) * c);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < DT; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) o_acc[i][r] *= alpha;
    }
    const float mc = m == -INFINITY ? 0.0f : m * c;
    bf16x8 p[2];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        float a = __builtin_amdgcn_exp2f(fmaf(s[j][r], c, -mc));
        float b = __builtin_amdgcn_exp2f(fmaf(s[j][r + 1], c, -mc));
        l += a + b;
        a -= __uint_as_float(__float_as_uint(a) & first);
        b -= __uint_as_float(__float_as_uint(b) & first);
        reinterpret_cast<unsigned*>(&p[j >> 1])[2 * (j & 1) + (r >> 1)] =
            __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
      }
#pragma unroll
    for (int i = 0; i < DT; i++) {
      o_acc[i] = kv8_mma16(kv8_wide(vr[i].x, vr[i].y, vs), p[0], o_acc[i]);
      o_acc[i] = kv8_mma16(kv8_wide(vr[i].z, vr[i].w, vs), p[1], o_acc[i]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) load_v(n + 1);
    __builtin_amdgcn_sched_barrier(0);
  }
  l = kv8_sum4(l);

  const int R = 2 * G;                       // second terms apart
  if (row_ok) {
    if (quad == 0 && !second) {
      ml_lds[wid][col][0] = m == -INFINITY ? m : m * sc.c;
      ml_lds[wid][col][1] = l;
    }
    float* mine = mo + (wid * R + (second ? G : 0) + col) * DP + 4 * quad;
#pragma unroll
    for (int i = 0; i < DT; i++)
      *reinterpret_cast<f4*>(mine + i * 16) = o_acc[i];
  }
  kv8_meet<D, SPLIT>(out, ws_o, ws_ml, mo, ml_lds, &flag, seq, kvh, part, parts, P, G,
                     n_kv, unit, out_stride, meet);
}
// Parts as over bf16 pages, by tiles of 64 keys where G <= 8. Few pairs are split later,
// from 14 tiles on: a wave's second and third tile cost less than the merge. Us, whole |
// in parts: 1 x 776 keys 7.0 | 7.3, 8 x 500 6.4 | 7.8, 1 x 2000 10.5 | 7.6, 8 x 2000 13.3 | 11.0.
// Up to 512 or 768 workgroups, with parts of 2 to 8 tiles, in place of 256 took as long or
// longer: 6 x 9-20 k 23.0 | 23.9 to 25.8, 4 x 8-30 k 34.7 | 36 to 37, 1 x 20 k 14.2 | 14.3 to 22.9.
// Many pairs gain nothing by parts here either: 128 sequences of 1-2 k keys 84 in one, 86
// in two, 88 in four; 48 of 12 heads of 64, up to 2000 keys, 20.8, 22.6, 22.4.
static PagedSplit kv8_split(long num_seqs, int n_kv, int G, long max_blocks) {
  PagedSplit x = paged_stream_split(num_seqs, n_kv, max_blocks);
  if (G > 8 || x.parts == 1) return x;
  const bool few = num_seqs * n_kv < 86;
  x.per = (x.per + 1) / 2;
  x.near = x.near >= 1 << 20 ? x.near : (x.near + 1) / 2;
  x.least = few ? 14 : (x.least + 1) / 2;
  x.parts = x.of((int)std::min<long>((max_blocks + 3) / 4, 1 << 20));
  return x;
}
int kv8_decode_parts(int num_seqs, int n_kv, int G, int max_blocks) {
  return kv8_split(num_seqs, n_kv, G, max_blocks).parts;
}

// ws_o, ws_ml: room for kv8_decode_parts() results per row and two counters a unit
void launch_kv8_decode(unsigned short* out, const unsigned short* q,
                       const unsigned char* k_cache, const unsigned char* v_cache,
                       const float* kv_scale, const int* block_tables,
                       const int* seq_lens, float* ws_ml, float* ws_o, float scale,
                       int num_seqs, int n_qheads, int n_kv, int D, int max_blocks,
                       int n_blocks, long q_stride, long out_stride,
                       hipStream_t stream) {
  if (num_seqs == 0) return;
  const PagedSplit split = kv8_split(num_seqs, n_kv, n_qheads / n_kv, max_blocks);
  PagedMeet meet;
  if (split.parts > 1)
    meet = paged_meet(ws_ml, (long)num_seqs * n_qheads, split.parts);
#define KV8_PICK(KERNEL)                                                       \
  (D == 128 ? (split.parts > 1 ? KERNEL<128, true> : KERNEL<128, false>)       \
            : (split.parts > 1 ? KERNEL<64, true> : KERNEL<64, false>))
  auto go = n_qheads / n_kv <= 8 ? KV8_PICK(kv8_decode16_kernel)
                                 : KV8_PICK(kv8_decode_kernel);
#undef KV8_PICK
  hipLaunchKernelGGL(go, dim3((unsigned)(num_seqs * n_kv * split.parts)), dim3(256),
                     0, stream, block_tables, seq_lens, n_qheads / n_kv, n_kv,
                     max_blocks, n_blocks, k_cache, v_cache,
                     reinterpret_cast<const float2*>(kv_scale), q, out, ws_o, ws_ml,
                     scale, q_stride, out_stride, split, meet);
}

}  // namespace xllm
