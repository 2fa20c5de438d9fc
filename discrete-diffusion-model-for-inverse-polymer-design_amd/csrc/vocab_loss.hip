// Cross entropy of the vocabulary head without keeping its logits (gfx950, bf16 MFMA).
//
//   z = h W^T,  loss = sum_i w_i (lse_i - z_{i, t_i}) / sum_i w_i,  lse_i = log sum_v exp z_iv
//   dz_iv = (g / sum w) w_i (exp(z_iv - lse_i) - [v = t_i]),   dh = dz W,  dW = dz^T h
//
// for hidden rows h [M, d] and head weights W [V, d]. Only rows with a weight (masked by the corruption and attended)
// are computed: they are first gathered, in order, into a compact matrix whose row count stays on the device.
//   forward:  tiles of z = Hc W^T reduce each row's maximum and sum of exponentials over 64 columns in registers; one
//             wave per row joins these pairs, adds the target's score (a dot product of its own) and the loss follows
//             in a fixed order: two runs give the same bits.
//   backward: piece by piece of the vocabulary, the tiles are computed again and leave w (p - onehot) in bf16 (values of
//             [-w, w], the common factor g / sum w is applied in fp32 where the products end), then
//             dh += dz W and dW = dz^T Hc. The last two read their operands along the summed axis through the
//             transposing LDS read, so that no transposed copy of anything is written. Sums over splits of a long axis
//             go to slabs of their own and are added in order.
// Bound by the matrix cores: 2 N V d flops forward and 6 N V d backward for N weighted rows.
#include "bd_common.h"
#include "bd_prof.h"
#include "bidiff.h"

namespace {

constexpr float VL_LOG2E = 1.44269504088896f, VL_LN2 = 0.69314718055995f;
constexpr int SCAN = 64;              // rows per workgroup of the gathering kernels

enum { VL_STATS = 0, VL_DLOG = 1, VL_SLAB = 2, VL_DW = 3 };

struct VlState {                      // what the forward leaves for the backward (device memory of the caller)
  int* head;                          // [0] weighted rows, [1] sum of weights (float bits)
  int *idx, *pos, *tgt;               // compact row -> row; row -> compact row or -1; target of a compact row
  float *w, *lse;                     // weight and log2-sum-exp2 of z * log2(e) of a compact row
  unsigned short* hc;                 // [m_pad, d] compact rows, zeros to the end of the last 64
  long long bytes;
};

__host__ __device__ inline long long vl_up(long long x, long long m) { return (x + m - 1) / m * m; }

VlState vl_state(void* base, long long M, int d) {
  char* p = (char*)base;
  const long long mp = vl_up(M, 256), r4 = vl_up(mp * 4, 256);
  VlState s;
  s.head = (int*)p; p += 256;
  s.idx = (int*)p; p += r4;
  s.pos = (int*)p; p += r4;
  s.tgt = (int*)p; p += r4;
  s.w = (float*)p; p += r4;
  s.lse = (float*)p; p += r4;
  s.hc = (unsigned short*)p; p += mp * d * 2;
  s.bytes = p - (char*)base;
  return s;
}

__device__ __forceinline__ float vl_weight(const unsigned char* ind, const long long* attn, long long m) {
  if (ind && !ind[m]) return 0.f;
  return attn ? (float)attn[m] : 1.f;
}

// weighted rows and sum of weights of each group of SCAN rows: one wave per group (32 768 rows: 3-5 us, a launch's latency)
__global__ __launch_bounds__(256) void vl_count_kernel(const unsigned char* __restrict__ ind, const long long* __restrict__ attn,
                                                       int* __restrict__ counts, float* __restrict__ sums, int M) {
  const int grp = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if ((long long)grp * SCAN >= M) return;
  const int row = grp * SCAN + lane;
  const float w = row < M ? vl_weight(ind, attn, row) : 0.f;
  const unsigned long long live = __ballot(w != 0.f);
  const float s = bd_wave_sum(w);
  if (lane == 0) { counts[grp] = __popcll(live); sums[grp] = s; }
}

// the group's weighted rows to their places: the counts of the groups before it are added up first (in order). Bound by
// memory behind that sum's latency (16 384 of 32 768 rows of 768 bytes: 25 MB in 8-9 us); a row's chunks are dealt to more
// workgroups from 512 values on.
__global__ __launch_bounds__(256) void vl_gather_kernel(const unsigned short* __restrict__ hidden, const long long* __restrict__ targets,
                                                        const unsigned char* __restrict__ ind, const long long* __restrict__ attn,
                                                        const int* __restrict__ counts, const float* __restrict__ sums, VlState st,
                                                        int M, int d, int V) {
  __shared__ int before[4], all[4], src[SCAN], here;
  __shared__ float wsum[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int groups = (M + SCAN - 1) / SCAN, grp = blockIdx.x;
  int nb = 0, na = 0;
  float ws = 0.f;
#pragma unroll 4
  for (int i = tid; i < groups; i += 256) {
    const int n = counts[i];
    na += n;
    if (i < grp) nb += n;
    ws += sums[i];
  }
  nb = bd_wave_sum_i(nb); na = bd_wave_sum_i(na); ws = bd_wave_sum(ws);
  if (lane == 0) { before[wave] = nb; all[wave] = na; wsum[wave] = ws; }
  __syncthreads();
  const int first = before[0] + before[1] + before[2] + before[3], total = all[0] + all[1] + all[2] + all[3];
  const bool lead = blockIdx.y == 0;
  if (wave == 0) {
    const int row = grp * SCAN + lane;
    const float w = row < M ? vl_weight(ind, attn, row) : 0.f;
    const unsigned long long live = __ballot(w != 0.f);
    const int at = __popcll(live & ((1ull << lane) - 1ull));
    if (lead && row < M) st.pos[row] = w != 0.f ? first + at : -1;
    if (w != 0.f) {
      src[at] = row;
    }
    if (lead && w != 0.f) {
      st.idx[first + at] = row;
      st.w[first + at] = w;
      const long long t = targets[row];
      st.tgt[first + at] = t >= 0 && t < V ? (int)t : -1;      // outside the vocabulary: the row's loss is NaN
    }
    if (lane == 0) here = __popcll(live);                  // (a place of its own: the other waves may still read before[])
    if (lead && grp == 0 && lane == 0) {
      st.head[0] = total;
      ((float*)st.head)[1] = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
    }
  }
  __syncthreads();
  // (the row's 16-byte chunks are dealt to the workgroups of a group, grid.y)
  const int n = here, per = d / 8, wide = (per + gridDim.y - 1) / gridDim.y, ch0 = wide * blockIdx.y, chn = min(wide, per - ch0);
  for (int i = tid; i < n * chn; i += 256) {
    const int r = i / chn, ch = ch0 + i - r * chn;
    *(u32x4*)(st.hc + (long long)(first + r) * d + 8 * ch) = *(const u32x4*)(hidden + (long long)src[r] * d + 8 * ch);
  }
  if (grp == groups - 1) {      // zeros behind the last row to the end of its 64: dW sums whole stages of rows (what a tile's
    const int tail = (int)vl_up(total, 64) - total;      // further rows hold reaches no row but their own)
    for (int i = tid; i < tail * chn; i += 256) {
      const int r = i / chn;
      *(u32x4*)(st.hc + (long long)(total + r) * d + 8 * (ch0 + i - r * chn)) = (u32x4){0u, 0u, 0u, 0u};
    }
  }
}

// =====================================================================================
// C[m, n] = sum_k A(m, k) B(n, k) on BM x BN tiles. AKC / BKC: the operand is stored along k (rows of K values) or, if not,
// along its own axis (row k holds the values of all m / n). MFMA operand order: n is the A side and m the B side, with n
// permuted inside 64 columns, so that a lane ends up with 2 x 8 consecutive n of one row m (columns 8 g and 32 + 8 g: the
// four lanes of a row store 64 consecutive bytes at a time). K is staged 64 at a time by LDS-DMA, two stages in turn (three
// or four stages of 32: 4-15 % slower). Bound by the matrix cores where the summed axis is long: 4096 x 2048 -> 65536 scores
// 746 us = 1.47 PFLOP/s (65 % of the cycles; the clock gives way under the load), dz 1.15, dh 1.3, dW 1.3; by the tiles'
// start and end at short ones: 16384 x 384 -> 803 0.4-0.6.
// =====================================================================================
// Splits of a product's summed axis: one workgroup per CU, four stages each at least. For dh the tiles follow the row count
// on the device, so the kernel and the one that adds the slabs up ask this themselves.
__host__ __device__ inline int vl_splits(long long tiles, long long k_tiles, int most) {
  long long n = tiles >= 256 ? 1 : tiles > 0 ? 256 / tiles : 1;
  if (n > k_tiles / 4) n = k_tiles / 4;
  return n < 1 ? 1 : n > most ? most : (int)n;
}
__device__ __forceinline__ int vl_dh_splits(int live, int bt, int d, int k, int most) {
  return vl_splits((long long)((live + bt - 1) / bt) * ((d + bt - 1) / bt), (k + 63) >> 6, most);
}

struct VlGemm {
  const unsigned short *A, *B;
  long long lda, ldb;
  const int* head;                    // weighted rows on the device
  int M, N, K;                        // capacities; m_live / k_live: M / K is the device's row count instead
  int n_rows;                         // rows of B that exist (BKC): columns behind them re-read the last one
  int m_live, k_live, n_split;
  int dh_split;                       // dh: n_split is the most, the kernel takes what the row count asks for
  unsigned short* dh;                 // dh from one piece and one split: written in bf16 to its rows, no slab
  const int* idx;
  const int* pos;                     // dh without a kernel behind it: the rows_all rows without weight are cleared here
  int rows_all;
  int v0, V;                          // VL_STATS, VL_DLOG: n is vocabulary column v0 + n, valid below V. VL_DW: m is
  const float *w, *lse;               // VL_DLOG
  const int* tgt;
  f32x2* pairs;                       // VL_STATS: [tile column][M] (maximum, sum) in base 2
  unsigned short* dlog;               // VL_DLOG: [M, ldo]
  float* slab;                        // VL_SLAB: [split][M][N]
  long long slab_stride, ldo;
  int add;                            // VL_SLAB: add to what the slab holds
  const float* gout;                  // VL_DW
  void* dw;                           // [V, N]: bf16, or fp32 that is added to
  int dw_f32;
};

typedef __attribute__((address_space(3))) void vl_lds;

// 16-byte chunk ch of a row: what 16 lanes read at a time covers every bank once
template <int R> __device__ __forceinline__ int vl_kc(int row, int ch) { return R * row + 16 * (ch ^ ((row >> 1) & 7)); }
template <int R> __device__ __forceinline__ int vl_mc(int row, int ch) { return R * row + 16 * (ch ^ ((row & 3) << 2)); }
__device__ __forceinline__ s16x4 vl_read_tr(const unsigned char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}
__device__ __forceinline__ bf16x8 vl_join(s16x4 a, s16x4 b) {
  union { struct { s16x4 a, b; } s; bf16x8 v; } u;
  u.s.a = a; u.s.b = b;
  return u.v;
}

// (the IEEE maximum: fmaxf would first quiet each product's result)
__device__ __forceinline__ float vl_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// (maximum, sum of 2^(x - maximum)) of two parts
__device__ __forceinline__ f32x2 vl_pair(f32x2 a, f32x2 b) {
  const float m = fmaxf(a[0], b[0]), ref = m == -INFINITY ? 0.f : m;
  return (f32x2){m, a[1] * __builtin_amdgcn_exp2f(a[0] - ref) + b[1] * __builtin_amdgcn_exp2f(b[0] - ref)};
}

// the columns a lane holds of a row (8 at o, 8 at o + 32), times f, in bf16
__device__ __forceinline__ void vl_store_bf16(unsigned short* o, const f32x4 (&a)[4], float f, bool first, bool second) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[2 * i] = bd_pack_bf16x2(f * a[2 * h + i][0], f * a[2 * h + i][1]);
      w[2 * i + 1] = bd_pack_bf16x2(f * a[2 * h + i][2], f * a[2 * h + i][3]);
    }
    if (h ? second : first) *(u32x4*)(o + 32 * h) = w;
  }
}

template <int BM, int BN, bool AKC, bool BKC, int EPI>
__global__ __launch_bounds__(2 * BN, 2) void vl_gemm_kernel(VlGemm p) {
  constexpr int WM = 2, WN = BN / 64, NW = WM * WN, TM = BM / WM / 16, TN = 4;
  constexpr int BK = 64, AHEAD = 2;
  constexpr int SA = BM * BK * 2, SB = BN * BK * 2, STAGE = SA + SB;      // bytes of a stage, either layout
  extern __shared__ __attribute__((aligned(1024))) unsigned char vl_smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int g = lane >> 4, c = lane & 15, q4 = c >> 2, p4 = c & 3;
  const int live = p.head[0];
  const int M = p.m_live ? min(live, p.M) : p.M, K = p.k_live ? min((live + 63) & ~63, p.K) : p.K;      // (whole stages of rows: zeros behind the last)
  if (EPI == VL_SLAB && p.pos) {                           // (every workgroup its share, with or without a tile)
    const int share = (p.rows_all + gridDim.x - 1) / gridDim.x, first = blockIdx.x * share, per = p.N / 8;
    for (int i = tid; i < min(share, p.rows_all - first) * per; i += 64 * NW) {
      const int row = first + i / per;
      if (p.pos[row] < 0) *(u32x4*)(p.dh + (long long)row * p.ldo + 8 * (i % per)) = (u32x4){0u, 0u, 0u, 0u};
    }
  }
  // tile list: groups of 8 tile rows, column by column inside a group; each XCD takes one contiguous part
  const int tiles_m = (M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
  const int n_split = p.dh_split ? vl_dh_splits(M, BM, p.N, p.K, p.n_split) : p.n_split, n_all = tiles_m * tiles_n * n_split;
  int tile;
  {
    const int xcd = blockIdx.x & 7, j = blockIdx.x >> 3, q = n_all >> 3, rr = n_all & 7;
    if (j >= q + (xcd < rr ? 1 : 0)) return;
    tile = (xcd < rr ? xcd * (q + 1) : rr * (q + 1) + (xcd - rr) * q) + j;
  }
  const int split = tile / (tiles_m * tiles_n);
  tile -= split * tiles_m * tiles_n;
  const int group = tile / (8 * tiles_n), rows_here = min(tiles_m - 8 * group, 8), in_group = tile - group * 8 * tiles_n;
  const int m0 = (8 * group + in_group % rows_here) * BM, n0 = (in_group / rows_here) * BN;
  const int kt_all = (K + 63) >> 6, kt_per = (kt_all + n_split - 1) / n_split;
  const int kt_beg = min(split * kt_per, kt_all), kt_end = min(kt_beg + kt_per, kt_all);

  // ---- staging: wave w sends pieces w, w + NW, ...; a lane's offset inside a stage's source is fixed but in a last
  //      stage that ends inside (summed axis along the rows), where rows past the end re-read the last one
  constexpr int PA = SA / 1024 / NW, PB = SB / 1024 / NW;
  auto off_a = [&](int j, int k0) -> unsigned {
    const int at = (wave + NW * j) * 1024 + lane * 16;
    if (AKC) {
      constexpr int R = 2 * BK;
      const int row = at / R, ch = (vl_kc<R>(row, (at % R) >> 4) - R * row) >> 4;
      return (unsigned)(((long long)(min(m0 + row, p.M - 1) - m0) * p.lda + 8 * ch) * 2);
    }
    constexpr int R = 2 * BM;
    const int row = at / R, ch = (vl_mc<R>(row, (at % R) >> 4) - R * row) >> 4;
    return (unsigned)(((long long)min(row, K - 1 - k0) * p.lda + min(m0 + 8 * ch, p.M - 8) - m0) * 2);
  };
  auto off_b = [&](int j, int k0) -> unsigned {
    const int at = (wave + NW * j) * 1024 + lane * 16;
    if (BKC) {
      constexpr int R = 2 * BK;
      const int rx = at / R, ch = (vl_kc<R>(rx, (at % R) >> 4) - R * rx) >> 4;
      const int i = rx & 15, tn = (rx >> 4) & 3, n = 64 * (rx >> 6) + 32 * (tn >> 1) + 8 * (i >> 2) + 4 * (tn & 1) + (i & 3);   // permuted
      return (unsigned)(((long long)(min(n0 + n, p.n_rows - 1) - n0) * p.ldb + 8 * ch) * 2);
    }
    constexpr int R = 2 * BN;
    const int row = at / R, ch = (vl_mc<R>(row, (at % R) >> 4) - R * row) >> 4;
    return (unsigned)(((long long)min(row, K - 1 - k0) * p.ldb + min(n0 + 8 * ch, p.N - 8) - n0) * 2);
  };
  unsigned va[PA], vb[PB];
#pragma unroll
  for (int j = 0; j < PA; ++j) va[j] = off_a(j, 0);
#pragma unroll
  for (int j = 0; j < PB; ++j) vb[j] = off_b(j, 0);
  const unsigned lds0 = (unsigned)(size_t)(vl_lds*)vl_smem;
  auto glds = [&](const unsigned char* src, unsigned vo, unsigned dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(vo), "s"(src) : "memory", "m0");
  };
  auto issue = [&](int kt, int buf) {
    const unsigned base = lds0 + buf * STAGE;
    const unsigned char* sa = (const unsigned char*)(AKC ? p.A + (long long)m0 * p.lda + (long long)BK * kt : p.A + (long long)BK * kt * p.lda + m0);
    const unsigned char* sb = (const unsigned char*)(BKC ? p.B + (long long)n0 * p.ldb + (long long)BK * kt : p.B + (long long)BK * kt * p.ldb + n0);
    const bool ragged = BK * kt + BK > K;
#pragma unroll
    for (int j = 0; j < PA; ++j) glds(sa, !AKC && ragged ? off_a(j, BK * kt) : va[j], base + (wave + NW * j) * 1024);
#pragma unroll
    for (int j = 0; j < PB; ++j) glds(sb, !BKC && ragged ? off_b(j, BK * kt) : vb[j], base + SA + (wave + NW * j) * 1024);
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  if (kt_beg < kt_end) issue(kt_beg, 0);
  int buf = 0;
  for (int kt = kt_beg; kt < kt_end; ++kt, buf ^= 1) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (kt + 1 < kt_end) issue(kt + 1, buf ^ 1);
    const unsigned char* const As = vl_smem + buf * STAGE;
    const unsigned char* const Bs = As + SA;
    auto load_x = [&](int kk, int tn) -> bf16x8 {
      if (BKC) return *(const bf16x8*)(Bs + vl_kc<2 * BK>(64 * wn + 16 * tn + c, 4 * kk + g));
      constexpr int R = 2 * BN;
      const int r0 = 32 * kk + 8 * g + q4, ch = 8 * wn + 4 * (tn >> 1) + p4;
      return vl_join(vl_read_tr(Bs + vl_mc<R>(r0, ch) + 8 * (tn & 1)), vl_read_tr(Bs + vl_mc<R>(r0 + 4, ch) + 8 * (tn & 1)));
    };
    auto load_y = [&](int kk, int tm) -> bf16x8 {
      if (AKC) return *(const bf16x8*)(As + vl_kc<2 * BK>(16 * TM * wm + 16 * tm + c, 4 * kk + g));
      constexpr int R = 2 * BM;
      const int r0 = 32 * kk + 8 * g + q4, ch = 2 * (TM * wm + tm) + (p4 >> 1);
      return vl_join(vl_read_tr(As + vl_mc<R>(r0, ch) + 8 * (p4 & 1)), vl_read_tr(As + vl_mc<R>(r0 + 4, ch) + 8 * (p4 & 1)));
    };
    // operand fragments are read AHEAD of their products, in this order (the compiler left alone reads one, waits for it and
    // multiplies: scores of 4096 x 2048 -> 65536 in 867 us instead of 746)
    constexpr int STEPS = BK / 32 * TM;
    bf16x8 x[2][TN], y[AHEAD];
#pragma unroll
    for (int tn = 0; tn < TN; ++tn) x[0][tn] = load_x(0, tn);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) y[i] = load_y(i / TM, i % TM);
    __builtin_amdgcn_sched_barrier(0x6);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int kk = i / TM, tm = i % TM;
#pragma unroll
      for (int tn = 0; tn < TN; ++tn) acc[tm][tn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[kk & 1][tn], y[i % AHEAD], acc[tm][tn], 0, 0, 0);
      if (i + AHEAD < STEPS) y[i % AHEAD] = load_y((i + AHEAD) / TM, (i + AHEAD) % TM);
      if (kk + 1 < BK / 32 && tm < TN) x[(kk + 1) & 1][tm] = load_x(kk + 1, tm);
      __builtin_amdgcn_sched_barrier(0x6);
    }
  }

  // ---- lane: row m0 + 16 (TM wm + tm) + c, columns nb + 32 (tn >> 1) + 4 (tn & 1) + j
  const int nb = n0 + 64 * wn + 8 * g;
  float coef = 0.f;
  if (EPI == VL_DW || EPI == VL_SLAB) {
    const float sw = ((const float*)p.head)[1];
    coef = sw > 0.f && p.gout ? p.gout[0] / sw : 0.f;
  }
  if (EPI == VL_STATS) {
    // each wave's 64 columns to a pair (maximum, sum) per row, joined over the tile's columns through LDS
    const bool whole = p.v0 + n0 + BN <= p.V;
    f32x2* const pl = (f32x2*)vl_smem;                     // [WN][BM]
    __syncthreads();
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) {
      if (!whole) {
#pragma unroll
        for (int tn = 0; tn < TN; ++tn)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (p.v0 + nb + 32 * (tn >> 1) + 4 * (tn & 1) + j >= p.V) acc[tm][tn][j] = -INFINITY;
      }
      float mx = -INFINITY, se = 0.f;
#pragma unroll
      for (int tn = 0; tn < TN; ++tn) mx = vl_max(vl_max(mx, vl_max(acc[tm][tn][0], acc[tm][tn][1])), vl_max(acc[tm][tn][2], acc[tm][tn][3]));
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float ref = mx == -INFINITY ? 0.f : mx * VL_LOG2E;
#pragma unroll
      for (int tn = 0; tn < TN; ++tn)
#pragma unroll
        for (int j = 0; j < 4; ++j) se += __builtin_amdgcn_exp2f(acc[tm][tn][j] * VL_LOG2E - ref);
      se += __shfl_xor(se, 16, 64);
      se += __shfl_xor(se, 32, 64);
      if (g == 0) pl[wn * BM + 16 * (TM * wm + tm) + c] = (f32x2){mx * VL_LOG2E, se};
    }
    __syncthreads();
    if (tid < BM && m0 + tid < M) {
      f32x2 x = pl[tid];
#pragma unroll
      for (int w = 1; w < WN; ++w) x = vl_pair(x, pl[w * BM + tid]);
      p.pairs[(long long)(n0 / BN) * p.M + m0 + tid] = x;
    }
    return;
  }
#pragma unroll
  for (int tm = 0; tm < TM; ++tm) {
    const int m = m0 + 16 * (TM * wm + tm) + c;
    if (EPI == VL_DLOG) {
      // (rows behind the last weighted one: zeros, they are summed over by dW's product)
      const bool in = m < M;
      const int tcol = in ? p.tgt[m] - p.v0 - nb : -1;
      const float lse = in ? p.lse[m] : INFINITY, w = in ? p.w[m] : 0.f;
#pragma unroll
      for (int tn = 0; tn < TN; ++tn)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int col = 32 * (tn >> 1) + 4 * (tn & 1) + j;
          const float pr = __builtin_amdgcn_exp2f(acc[tm][tn][j] * VL_LOG2E - lse);
          acc[tm][tn][j] = w * (col == tcol ? pr - 1.f : pr);
        }
      if (p.v0 + n0 + BN > p.V || !in) {
#pragma unroll
        for (int tn = 0; tn < TN; ++tn)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (!in || p.v0 + nb + 32 * (tn >> 1) + 4 * (tn & 1) + j >= p.V) acc[tm][tn][j] = 0.f;
      }
      vl_store_bf16(p.dlog + (long long)m * p.ldo + nb, acc[tm], 1.f, nb < p.N, nb + 32 < p.N);
    } else if (EPI == VL_SLAB) {
      if (m >= M) continue;
      if (p.dh && n_split == 1) {
        vl_store_bf16(p.dh + (long long)p.idx[m] * p.ldo + nb, acc[tm], coef, nb < p.N, nb + 32 < p.N);
        continue;
      }
      float* o = p.slab + split * p.slab_stride + (long long)m * p.ldo + nb;
#pragma unroll
      for (int tn = 0; tn < TN; ++tn) {
        const int col = 32 * (tn >> 1) + 4 * (tn & 1);
        if (nb + col >= p.N) continue;
        f32x4 x = acc[tm][tn];
        if (p.add) {
          const f32x4 y = *(const f32x4*)(o + col);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] += y[j];
        }
        *(f32x4*)(o + col) = x;
      }
    } else {
      if (p.v0 + m >= p.V) continue;
      const long long at = (long long)(p.v0 + m) * p.ldo + nb;
      if (!p.dw_f32) {
        vl_store_bf16((unsigned short*)p.dw + at, acc[tm], coef, nb < p.N, nb + 32 < p.N);
        continue;
      }
      float* o = (float*)p.dw + at;
#pragma unroll
      for (int tn = 0; tn < TN; ++tn) {
        const int col = 32 * (tn >> 1) + 4 * (tn & 1);
        if (nb + col >= p.N) continue;
        f32x4 y = *(const f32x4*)(o + col);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] += coef * acc[tm][tn][j];
        *(f32x4*)(o + col) = y;
      }
    }
  }
}

// one wave per weighted row: joins the row's pairs and computes the target's score; rowloss[r] = w (lse - z_t). Latency of
// two dependent reads a row (16 384 rows of 384: 7 us)
__global__ __launch_bounds__(256) void vl_join_kernel(VlState st, const unsigned short* __restrict__ weight, const f32x2* __restrict__ pairs,
                                                      float* __restrict__ rowloss, int cap, int blocks, int d) {
  const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= st.head[0]) return;
  f32x2 ms = {-INFINITY, 0.f};
  for (int i = lane; i < blocks; i += 64) ms = vl_pair(ms, pairs[(long long)i * cap + row]);
  const float m = ms[0];
  float s = ms[1];
  const float mm = bd_wave_max(m);
  const float ref = mm == -INFINITY ? 0.f : mm;
  s = bd_wave_sum(s * __builtin_amdgcn_exp2f(m - ref));
  const float lse = ref + __log2f(s);
  const int t = st.tgt[row];
  float z = 0.f;
  if (t >= 0) {
    const unsigned short *x = st.hc + (long long)row * d, *y = weight + (long long)t * d;
    for (int i = 8 * lane; i < d; i += 512) {
      const bf16x8 a = *(const bf16x8*)(x + i), b = *(const bf16x8*)(y + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) z += (float)a[e] * (float)b[e];
    }
  }
  z = bd_wave_sum(z);
  if (lane == 0) {
    st.lse[row] = lse;
    rowloss[row] = t >= 0 ? st.w[row] * (lse * VL_LN2 - z) : __uint_as_float(0x7fc00000u);
  }
}

// loss = sum rowloss / sum w, in a fixed order; an exact zero without a weighted row (16 384 rows: 4 us, one workgroup's
// latency)
__global__ __launch_bounds__(1024) void vl_finish_kernel(VlState st, const float* __restrict__ rowloss, float* __restrict__ loss) {
  __shared__ float part[16];
  const int n = st.head[0];
  float s = 0.f;
#pragma unroll 4
  for (int i = 4 * threadIdx.x; i < n; i += 4096) {        // (rows behind the last: whatever is there, not added)
    const f32x4 x = *(const f32x4*)(rowloss + i);
    s += (x[0] + (i + 1 < n ? x[1] : 0.f)) + ((i + 2 < n ? x[2] : 0.f) + (i + 3 < n ? x[3] : 0.f));
  }
  s = bd_wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
    for (int i = 0; i < 16; ++i) t += part[i];
    const float sw = ((const float*)st.head)[1];
    loss[0] = sw > 0.f ? t / sw : 0.f;
  }
}

// dhidden rows from the slabs (added in order), zeros at rows without a weight. Bound by memory (3001 x 768, 8 slabs: 12 us)
__global__ __launch_bounds__(256) void vl_dh_kernel(VlState st, const float* __restrict__ slab, long long slab_stride, int most, int bt, int k,
                                                    int pieces, const float* __restrict__ gout, unsigned short* __restrict__ dh, int M, int d) {
  const int per = d / 8;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)M * per) return;
  const int row = (int)(i / per), ch = (int)(i - (long long)row * per);
  const int at = st.pos[row];
  u32x4 o = {0u, 0u, 0u, 0u};
  if (at >= 0) {
    const int n_slab = vl_dh_splits(st.head[0], bt, d, k, most);
    if (n_slab == 1 && pieces == 1) return;                // the product wrote the row itself
    const float sw = ((const float*)st.head)[1];
    const float coef = sw > 0.f ? gout[0] / sw : 0.f;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < n_slab; ++s) {
      const float* p = slab + s * slab_stride + (long long)at * d + 8 * ch;
      const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] += a[e]; v[4 + e] += b[e]; }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = bd_pack_bf16x2(coef * v[2 * e], coef * v[2 * e + 1]);
  }
  *(u32x4*)(dh + (long long)row * d + 8 * ch) = o;
}

// dW rows v0 .. v0 + rows from the slabs of their splits: 32 units of 8 values a workgroup, each added up by eight threads that
// take every eighth slab, then in order. Bound by memory (803 x 384, 10 slabs: 4.1 us; one thread a unit 4.6) or latency
// (39 x 64, 64 slabs: 3.6 us; one thread a unit 16.7)
__global__ __launch_bounds__(256) void vl_dw_kernel(VlState st, const float* __restrict__ slab, long long slab_stride, int n_slab,
                                                    const float* __restrict__ gout, void* __restrict__ dw, int dw_f32, int v0, int rows, int d) {
  __shared__ float part[7][32][9];
  const int tid = threadIdx.x, unit = tid & 31, from = tid >> 5;
  const long long i = (long long)blockIdx.x * 32 + unit, all = (long long)rows * (d / 8);
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (i < all) {
#pragma unroll 4
    for (int s = from; s < n_slab; s += 8) {
      const float* p = slab + s * slab_stride + 8 * i;
      const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] += a[e]; v[4 + e] += b[e]; }
    }
  }
  if (from > 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) part[from - 1][unit][e] = v[e];
  }
  __syncthreads();
  if (from > 0 || i >= all) return;
#pragma unroll
  for (int f = 0; f < 7; ++f)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += part[f][unit][e];
  const float sw = ((const float*)st.head)[1];
  const float coef = sw > 0.f ? gout[0] / sw : 0.f;
  const long long at = (long long)v0 * d + 8 * i;
  if (dw_f32) {
    float* o = (float*)dw + at;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] += coef * v[e];
  } else {
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = bd_pack_bf16x2(coef * v[2 * e], coef * v[2 * e + 1]);
    *(u32x4*)((unsigned short*)dw + at) = o;
  }
}

// =====================================================================================
// Forward for a vocabulary of at most 64 classes: 16 rows a workgroup, straight from where they lie (they are gathered
// beside it only where a backward follows; it then leaves their log-sum-exps at their compact places). The waves share the
// rows and deal the hidden size among them (32 values in turn; the small call is bound by latency: every load of a wave is
// asked for before its first product); their scores meet in LDS, where 16 threads finish a row. Transposed products (z^T = W
// h^T): a lane's scores are one row's. Then the workgroups' sums are added in order. Measured, hidden size 384, half of the
// rows weighted, this / gathered rows and tiles, without a backward, us: 512 rows, 39 classes 8.6 / 23; 32768 rows, 39
// classes 18 / 36 (beside the gathering for a backward 18 / 21). At 128 classes it is 34 / 36 and 37 / 21: every workgroup
// reads the head's rows again.
// =====================================================================================
constexpr int VL_NARROW = 64, VL_NROWS = 16;
__global__ __launch_bounds__(256, 2) void vl_narrow_kernel(const unsigned short* __restrict__ hidden, const unsigned short* __restrict__ weight,
                                                           const long long* __restrict__ targets, const unsigned char* __restrict__ ind,
                                                           const long long* __restrict__ attn, f32x2* __restrict__ sums, VlState st, int M, int d, int V) {
  constexpr int NT = VL_NARROW / 16, LD = VL_NARROW + 4, STEPS = 3;
  __shared__ __attribute__((aligned(16))) float z[4][VL_NROWS][LD];
  __shared__ f32x2 part[VL_NROWS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const int row = blockIdx.x * VL_NROWS + c;
  const float w = row < M ? vl_weight(ind, attn, row) : 0.f;
  if (!__any(w != 0.f)) {
    if (tid == 0) sums[blockIdx.x] = (f32x2){0.f, 0.f};
    return;
  }
  const unsigned short* x = hidden + (long long)row * d + 8 * g;
  const unsigned short* y = weight + (long long)min(c, V - 1) * d + 8 * g;
  f32x4 acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int steps = d / 32;
  for (int k0 = wave; k0 < steps; k0 += 4 * STEPS) {
    bf16x8 xf[STEPS] = {}, yf[STEPS][NT] = {};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int k = k0 + 4 * i;
      if (k >= steps) continue;
      if (w != 0.f) xf[i] = *(const bf16x8*)(x + 32 * k);
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (16 * j < V) yf[i][j] = *(const bf16x8*)(y + (long long)(min(16 * j + c, V - 1) - min(c, V - 1)) * d + 32 * k);
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(yf[i][j], xf[i], acc[j], 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) *(f32x4*)&z[wave][c][16 * j + 4 * g] = acc[j];    // row c, classes 16 j + 4 g ..
  __syncthreads();
  const int r = tid >> 4, v0 = tid & 15, rr = blockIdx.x * VL_NROWS + r;
  const float wr = rr < M ? vl_weight(ind, attn, rr) : 0.f;
  const long long t = wr != 0.f ? targets[rr] : 0;
  float s[NT], mx = -INFINITY, zt = 0.f;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int v = 16 * j + v0;
    s[j] = (z[0][r][v] + z[1][r][v]) + (z[2][r][v] + z[3][r][v]);
    if (v < V) mx = fmaxf(mx, s[j]);
    if (v == t) zt = s[j];
  }
#pragma unroll
  for (int i = 1; i < 16; i *= 2) mx = fmaxf(mx, __shfl_xor(mx, i, 64));
  const float ref = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NT; ++j)
    if (16 * j + v0 < V) sum += __builtin_amdgcn_exp2f((s[j] - ref) * VL_LOG2E);
#pragma unroll
  for (int i = 1; i < 16; i *= 2) { sum += __shfl_xor(sum, i, 64); zt += __shfl_xor(zt, i, 64); }
  if (v0 == 0) {
    const float lse = ref * VL_LOG2E + __log2f(sum);
    if (st.head && wr != 0.f) st.lse[st.pos[rr]] = lse;
    const float l = t >= 0 && t < V ? wr * (lse * VL_LN2 - zt) : __uint_as_float(0x7fc00000u);   // outside the vocabulary: NaN
    part[r] = (f32x2){wr != 0.f ? l : 0.f, wr};
  }
  __syncthreads();
  if (tid == 0) {
    f32x2 a = {0.f, 0.f};
    for (int i = 0; i < VL_NROWS; ++i) { a[0] += part[i][0]; a[1] += part[i][1]; }
    sums[blockIdx.x] = a;
  }
}

__global__ __launch_bounds__(1024) void vl_narrow_finish_kernel(const f32x2* __restrict__ sums, int n, float* __restrict__ loss) {
  __shared__ f32x2 part[16];
  f32x2 a = {0.f, 0.f};
  for (int i = threadIdx.x; i < n; i += 1024) { const f32x2 x = sums[i]; a[0] += x[0]; a[1] += x[1]; }
  a = (f32x2){bd_wave_sum(a[0]), bd_wave_sum(a[1])};
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    f32x2 t = {0.f, 0.f};
    for (int i = 0; i < 16; ++i) { t[0] += part[i][0]; t[1] += part[i][1]; }
    loss[0] = t[1] > 0.f ? t[0] / t[1] : 0.f;
  }
}

// ---------------------------------------------------------------------------------------------- host side
struct VlPlan {
  long long m_pad;
  int piece, n_pieces;                // vocabulary columns per backward piece
  int big_s, big_z, big_h, big_w;     // 256 x 256 tiles for the scores, dz, dh, dW (else 128 x 128)
  int split_h, split_w;               // splits of dh's product over the piece (at most), of dW's over the rows
  long long slab_h, slab_w;           // floats of one slab
  bool dh_alone;                      // one piece, one split: the product writes every row of dh, no slab to add up
  long long fwd_bytes;
};

// dz of one piece: what stays near the card's last-level cache (a piece has 256 columns at least: from 2^19 rows on it is
// 512 bytes a row)
constexpr long long VL_PIECE_BYTES = 256ll << 20;

VlPlan vl_plan(long long M, int d, int V) {
  VlPlan p;
  p.m_pad = vl_up(M, 256);
  // Tile sizes, each measured both ways (256 x 256 / 128 x 128, us; half of the rows weighted): the larger tile reads less LDS
  // per product but leaves one workgroup on a CU, whose start and end nothing hides, and wastes more at ragged edges and
  // in a last round of few tiles.
  //                     scores      scores again, to dz   dh (with the sum of its splits)   dW (with the sum of its splits)
  //   8192 x 2048 -> 65536  804 / 1011   979 / 1076   917 / 987   899 / 951
  //   8192 x 1024 -> 65536  420 / 504    567 / 610    494 / 684   433 / 458
  //   2000 x 1024 -> 65536  130 / 136    155 / 137    141 / 178   137 / 147
  //   4096 x 512 -> 32000    73 / 76      97 / 92      79 / 91     64 / 67
  //   3001 x 768 -> 32003    92 / 88     114 / 104     93 / 120   102 / 87
  //   8192 x 768 -> 8192     48 / 53      60 / 62      67 / 86     74 / 57
  //   32768 x 384 -> 4096    58 / 64      82 / 80      76 / 66     74 / 90
  //   32768 x 384 -> 803     17 / 18      25 / 25      37 / 25     39 / 28
  //   8192 x 4096 -> 2048    88 / 63      96 / 64      73 / 83     82 / 66
  // The rules below follow the column but for a few per cent: 3001 x 768 -> 32003 takes the larger tile for its scores (92,
  // not 88), 32768 x 384 -> 803 sits on that rule's border (17 / 18 is noise).
  const long long tiles_z = (p.m_pad / 256) * ((V + 255) / 256), tiles_w = (long long)((V + 255) / 256) * ((d + 255) / 256);
  p.big_s = tiles_z >= 512;
  p.big_z = d >= 1024 && tiles_z >= 4096;
  p.big_h = V >= 2048 && (d % 256 == 0 || d >= 768);
  p.big_w = 10 * tiles_w >= 9 * vl_up(tiles_w, 256);      // whole rounds of the CUs
  const int bh = p.big_h ? 256 : 128, bw = p.big_w ? 256 : 128;
  long long piece = VL_PIECE_BYTES / 2 / p.m_pad / 256 * 256;
  if (piece < 256) piece = 256;
  const long long v_pad = vl_up(V, 256);
  if (piece > v_pad) piece = v_pad;
  p.n_pieces = (int)((v_pad + piece - 1) / piece);
  p.piece = (int)vl_up((v_pad + p.n_pieces - 1) / p.n_pieces, 256);
  // (a quarter of the rows may carry weight: then dh has so many fewer tiles. At most 512 MB of slabs, or a single one.)
  p.slab_h = p.m_pad * d;
  p.split_h = vl_splits((vl_up(M, bh) / bh + 3) / 4 * (vl_up(d, bh) / bh), p.piece / 64, 64);
  while (p.split_h > 1 && p.split_h * p.slab_h * 4 > (512ll << 20)) --p.split_h;
  p.dh_alone = p.n_pieces == 1 && p.split_h == 1;
  // (fewer than 256 tiles times splits of a tile: at most 64 MB of slabs)
  p.split_w = vl_splits(vl_up(p.piece, bw) / bw * (vl_up(d, bw) / bw), p.m_pad / 64, 64);
  p.slab_w = (long long)p.piece * d;
  const long long groups = (M + SCAN - 1) / SCAN;
  p.fwd_bytes = vl_up(groups * 4, 256) * 2 + vl_up(p.m_pad * 4, 256) + (v_pad / 128) * p.m_pad * 8;
  return p;
}

// floats of all slabs of dh, of dW
long long vl_dh_slabs(const VlPlan& p) { return p.dh_alone ? 0 : p.split_h * p.slab_h; }
long long vl_dw_slabs(const VlPlan& p) { return p.split_w > 1 ? p.split_w * p.slab_w : 0; }
long long vl_bwd_bytes(const VlPlan& p, bool dh, bool dw) {
  return p.m_pad * p.piece * 2 + ((dh ? vl_dh_slabs(p) : 0) + (dw ? vl_dw_slabs(p) : 0)) * 4;
}

template <int BT, bool AKC, bool BKC, int EPI>
void vl_launch_tile(const VlGemm& p, hipStream_t s) {
  constexpr int LDS = 2 * (BT + BT) * 128;
  const long long n = vl_up(p.M, BT) / BT * (vl_up(p.N, BT) / BT) * p.n_split;
  BD_SET_MAX_LDS((vl_gemm_kernel<BT, BT, AKC, BKC, EPI>), LDS);
  hipLaunchKernelGGL((vl_gemm_kernel<BT, BT, AKC, BKC, EPI>), dim3((unsigned)vl_up(n, 8)), dim3(2 * BT), LDS, s, p);
}
template <bool AKC, bool BKC, int EPI>
void vl_launch(int big, const VlGemm& p, hipStream_t s) {
  if (big) vl_launch_tile<256, AKC, BKC, EPI>(p, s);
  else vl_launch_tile<128, AKC, BKC, EPI>(p, s);
}

int vl_check(long long M, int d, int V, const char* what) {
  BD_REQUIRE(M > 0 && V > 0 && d > 0, "%s: empty shape", what);
  BD_REQUIRE(d % 64 == 0, "%s: the hidden size %d must be a multiple of 64", what, d);
  BD_REQUIRE(M < (1ll << 24) && V < (1 << 28) && d <= 65536, "%s: too many rows, columns or classes", what);
  return BD_OK;
}

}  // namespace

extern "C" long long bd_linear_ce_state_bytes(long long M, int d) { return M > 0 && d > 0 ? vl_state(nullptr, M, d).bytes : -1; }

extern "C" long long bd_linear_ce_workspace_bytes(long long M, int d, int V, int kind) {
  if (M <= 0 || d <= 0 || V <= 0) return -1;
  if (kind == 2 && V <= VL_NARROW) return vl_up(vl_up(M, VL_NROWS) / VL_NROWS * 8, 256);
  const VlPlan p = vl_plan(M, d, V);
  if (kind == 1 || kind == 3 || kind == 4) return vl_bwd_bytes(p, kind != 3, kind != 4);
  return p.fwd_bytes + (kind == 2 ? bd_linear_ce_state_bytes(M, d) : 0);
}

extern "C" int bd_linear_ce_fwd(const void* hidden, const void* weight, const long long* targets, const unsigned char* indicator,
                                const long long* attention_mask, float* loss, long long M, int d, int V, void* state, long long state_bytes,
                                void* workspace, long long workspace_bytes, void* stream) {
  const int rc = vl_check(M, d, V, "bd_linear_ce_fwd");
  if (rc != BD_OK) return rc;
  BD_REQUIRE(hidden && weight && targets && loss && workspace, "bd_linear_ce_fwd: null operand");
  BD_REQUIRE((((uintptr_t)hidden | (uintptr_t)weight | (uintptr_t)state | (uintptr_t)workspace) & 15) == 0,
             "bd_linear_ce_fwd: operands must be 16-byte aligned");
  const long long need = bd_linear_ce_workspace_bytes(M, d, V, state ? 0 : 2);
  BD_REQUIRE(!state || state_bytes >= bd_linear_ce_state_bytes(M, d), "bd_linear_ce_fwd: the state must hold %lld bytes",
             bd_linear_ce_state_bytes(M, d));
  BD_REQUIRE(workspace_bytes >= need, "bd_linear_ce_fwd: the workspace must hold %lld bytes", need);
  hipStream_t s = (hipStream_t)stream;
  bd_prof_scope prof(stream, 2.0 * M * (double)V * d, BD_PROF_GEMM);
  const bool narrow = V <= VL_NARROW;
  const VlPlan pl = vl_plan(M, d, V);
  const VlState st = state ? vl_state(state, M, d) : narrow ? VlState{} : vl_state((char*)workspace + pl.fwd_bytes, M, d);
  const int groups = (int)((M + SCAN - 1) / SCAN);
  char* w = (char*)workspace;
  int* counts = (int*)w; w += vl_up(groups * 4ll, 256);
  float* sums = (float*)w; w += vl_up(groups * 4ll, 256);
  float* rowloss = (float*)w; w += vl_up(pl.m_pad * 4, 256);
  f32x2* pairs = (f32x2*)w;
  if (st.head) {
    hipLaunchKernelGGL(vl_count_kernel, dim3((groups + 3) / 4), dim3(256), 0, s, indicator, attention_mask, counts, sums, (int)M);
    hipLaunchKernelGGL(vl_gather_kernel, dim3(groups, (d + 511) / 512), dim3(256), 0, s, (const unsigned short*)hidden, targets, indicator,
                       attention_mask, counts, sums, st, (int)M, d, V);
  }
  if (narrow) {
    const int blocks = (int)(vl_up(M, VL_NROWS) / VL_NROWS);
    f32x2* parts = state ? pairs : (f32x2*)workspace;
    hipLaunchKernelGGL(vl_narrow_kernel, dim3(blocks), dim3(256), 0, s, (const unsigned short*)hidden, (const unsigned short*)weight, targets, indicator,
                       attention_mask, parts, st, (int)M, d, V);
    hipLaunchKernelGGL(vl_narrow_finish_kernel, dim3(1), dim3(1024), 0, s, parts, blocks, loss);
    return bd_check_launch("bd_linear_ce_fwd");
  }
  const int bz = pl.big_s ? 256 : 128;
  VlGemm p = {};
  p.A = st.hc; p.lda = d; p.B = (const unsigned short*)weight; p.ldb = d; p.head = st.head;
  p.M = (int)pl.m_pad; p.N = V; p.n_rows = V; p.K = d; p.m_live = 1; p.n_split = 1; p.V = V; p.pairs = pairs;
  vl_launch<true, true, VL_STATS>(pl.big_s, p, s);
  hipLaunchKernelGGL(vl_join_kernel, dim3((unsigned)((M + 3) / 4)), dim3(256), 0, s, st, (const unsigned short*)weight, pairs, rowloss,
                     (int)pl.m_pad, (V + bz - 1) / bz, d);
  hipLaunchKernelGGL(vl_finish_kernel, dim3(1), dim3(1024), 0, s, st, rowloss, loss);
  return bd_check_launch("bd_linear_ce_fwd");
}

extern "C" int bd_linear_ce_bwd(const void* weight, const float* grad_out, void* dhidden, void* dweight, int dweight_dtype, long long M, int d,
                                int V, const void* state, long long state_bytes, void* workspace, long long workspace_bytes, void* stream) {
  const int rc = vl_check(M, d, V, "bd_linear_ce_bwd");
  if (rc != BD_OK) return rc;
  BD_REQUIRE(weight && grad_out && (dhidden || dweight) && state && workspace, "bd_linear_ce_bwd: null operand");
  BD_REQUIRE((((uintptr_t)weight | (uintptr_t)dhidden | (uintptr_t)dweight | (uintptr_t)state | (uintptr_t)workspace) & 15) == 0,
             "bd_linear_ce_bwd: operands must be 16-byte aligned");
  BD_REQUIRE(dweight_dtype == BD_DTYPE_BF16 || dweight_dtype == BD_DTYPE_F32, "bd_linear_ce_bwd: dweight is neither bf16 nor fp32");
  const VlPlan pl = vl_plan(M, d, V);
  BD_REQUIRE(state_bytes >= bd_linear_ce_state_bytes(M, d), "bd_linear_ce_bwd: the state must hold %lld bytes", bd_linear_ce_state_bytes(M, d));
  const long long need = vl_bwd_bytes(pl, dhidden != nullptr, dweight != nullptr);
  BD_REQUIRE(workspace_bytes >= need, "bd_linear_ce_bwd: the workspace must hold %lld bytes", need);
  hipStream_t s = (hipStream_t)stream;
  const VlState st = vl_state((void*)state, M, d);
  unsigned short* dlog = (unsigned short*)workspace;
  float* slab_h = (float*)((char*)workspace + pl.m_pad * pl.piece * 2);
  float* slab_w = slab_h + (dhidden ? vl_dh_slabs(pl) : 0);
  bd_prof_scope prof(stream, 6.0 * M * (double)V * d, BD_PROF_GEMM);
  for (int i = 0; i < pl.n_pieces; ++i) {
    const int v0 = i * pl.piece, n = min(pl.piece, (int)vl_up(V - v0, 64));       // columns of the piece, whole 64s
    if (v0 >= V) break;
    const unsigned short* wp = (const unsigned short*)weight + (long long)v0 * d;
    VlGemm p = {};
    p.A = st.hc; p.lda = d; p.B = wp; p.ldb = d; p.head = st.head; p.M = (int)pl.m_pad; p.N = n; p.n_rows = min(n, V - v0); p.K = d; p.m_live = 1; p.n_split = 1;
    p.v0 = v0; p.V = V; p.w = st.w; p.lse = st.lse; p.tgt = st.tgt; p.dlog = dlog; p.ldo = pl.piece;
    vl_launch<true, true, VL_DLOG>(pl.big_z, p, s);
    if (dhidden) {
      p = VlGemm();
      p.A = dlog; p.lda = pl.piece; p.B = wp; p.ldb = d; p.head = st.head; p.M = (int)pl.m_pad; p.N = d; p.K = min(n, V - v0); p.m_live = 1;
      p.n_split = pl.split_h; p.dh_split = 1; p.slab = slab_h; p.slab_stride = pl.slab_h; p.ldo = d; p.add = i > 0;
      if (pl.n_pieces == 1) { p.dh = (unsigned short*)dhidden; p.idx = st.idx; p.gout = grad_out; }
      if (pl.dh_alone) { p.pos = st.pos; p.rows_all = (int)M; }
      vl_launch<true, false, VL_SLAB>(pl.big_h, p, s);
    }
    if (dweight) {
      p = VlGemm();
      p.A = dlog; p.lda = pl.piece; p.B = st.hc; p.ldb = d; p.head = st.head; p.M = n; p.N = d; p.K = (int)pl.m_pad; p.k_live = 1;
      p.n_split = pl.split_w; p.v0 = v0; p.V = V; p.ldo = d;
      if (pl.split_w > 1) {
        p.slab = slab_w; p.slab_stride = pl.slab_w;
        vl_launch<false, false, VL_SLAB>(pl.big_w, p, s);
        const int rows = min(n, V - v0);
        const long long items = (long long)rows * (d / 8);
        hipLaunchKernelGGL(vl_dw_kernel, dim3((unsigned)((items + 31) / 32)), dim3(256), 0, s, st, slab_w, pl.slab_w, pl.split_w, grad_out,
                           dweight, dweight_dtype == BD_DTYPE_F32, v0, rows, d);
      } else {
        p.gout = grad_out; p.dw = dweight; p.dw_f32 = dweight_dtype == BD_DTYPE_F32;
        vl_launch<false, false, VL_DW>(pl.big_w, p, s);
      }
    }
  }
  if (dhidden && !pl.dh_alone)
    hipLaunchKernelGGL(vl_dh_kernel, dim3((unsigned)((M * (d / 8) + 255) / 256)), dim3(256), 0, s, st, slab_h, pl.slab_h, pl.split_h,
                       pl.big_h ? 256 : 128, min(pl.piece, V), pl.n_pieces, grad_out, (unsigned short*)dhidden, (int)M, d);
  return bd_check_launch("bd_linear_ce_bwd");
}
