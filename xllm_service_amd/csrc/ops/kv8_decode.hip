// Paged attention of decoded rows over a cache held in 8 bits (kv8.h): bf16 in and out.
//
// For one (sequence, key head) the G query heads (G <= 16) are the columns of
// S^T = K Q^T and of O^T += V^T P^T on 32x32x16 products (layouts: mfma_rows.h). A
// tile is 32 keys, two pages. What the A operands want of a lane lies side by side in
// the pages, so a tile goes from memory to registers in 16 B a lane and is converted
// there, the scale of its page in the same instruction: no LDS, no transposes, no
// barrier in the loop.
//
//   keys     row m of A is key 4 (m >> 3) + (m & 3) of page (m >> 2) & 1: then the 16
//            scores that lane half h holds of a column are those of page h, in order
//   values   lane half h gives page h: its 16 bytes of a channel are the operands
//            of both steps that its 16 weights want
//   channels of a key are summed in the order of its 16 B chunks, h taking every
//            second one, queries likewise
//
// Weights have two bf16 terms (16 bits), the second ones in the columns that 16 heads
// leave (paged_stream.h). Waves have tiles of their own and meet in LDS at the end;
// long sequences are split over workgroups, the last of which merges (paged_merge.h).
#include "kv8.h"
#include "paged_stream.h"

namespace xllm {

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
  __shared__ float ml_lds[NW][32][2];
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
  Tile now, next;
  if (i0 < n_tiles) load(0, now);
  for (int t = i0, n = 0; t < n_tiles; t += step, n++) {
    if (t + step < n_tiles) {
      if (n + 1 - tb == 32) {
        tb += 32;
        look_up(tb);
      }
      load(n + 1, next);
    }
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
    now = next;
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
  if (!SPLIT || parts == 1 || !paged_last(meet.count + unit, parts, &flag)) return;
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

static PagedSplit kv8_split(long num_seqs, int n_kv, long max_blocks) {
  return paged_stream_split(num_seqs, n_kv, max_blocks);
}
int kv8_decode_parts(int num_seqs, int n_kv, int max_blocks) {
  return kv8_split(num_seqs, n_kv, max_blocks).parts;
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
  const PagedSplit split = kv8_split(num_seqs, n_kv, max_blocks);
  PagedMeet meet;
  if (split.parts > 1)
    meet = paged_meet(ws_ml, (long)num_seqs * n_qheads, split.parts);
  auto go = D == 128 ? (split.parts > 1 ? kv8_decode_kernel<128, true>
                                        : kv8_decode_kernel<128, false>)
                     : (split.parts > 1 ? kv8_decode_kernel<64, true>
                                        : kv8_decode_kernel<64, false>);
  hipLaunchKernelGGL(go, dim3((unsigned)(num_seqs * n_kv * split.parts)), dim3(256),
                     0, stream, block_tables, seq_lens, n_qheads / n_kv, n_kv,
                     max_blocks, n_blocks, k_cache, v_cache,
                     reinterpret_cast<const float2*>(kv_scale), q, out, ws_o, ws_ml,
                     scale, q_stride, out_stride, split, meet);
}

}  // namespace xllm
