// Differential attention (gfx950, bf16 MFMA): the difference of two softmax maps over one set of values.
//
//   out_i = sum_j (P1_ij - lam_i P2_ij) v_j,   Pm_ij = softmax_j(scale * q_im . k_jm) over the visible keys,
//
// for H heads of two maps each (query / key heads 2 h and 2 h + 1, head size D) and values of width E = 2 D; Hkv key /
// value heads are shared by H / Hkv heads each. A query without a visible key gives a zero row. Backward, with
// dP_ij = dO_i . v_j and delta_m = sum_j Pm_ij dP_ij:
//
//   dV_j = sum_i (P1 - lam P2)_ij dO_i          dlam_i = -delta_2
//   dS1 = P1 (dP - delta_1), dS2 = -lam P2 (dP - delta_2), dQm = scale dSm Km, dKm = scale dSm^T Qm
//
// Queries are handled as SLOTS: slot s of a sequence and key head is (row s / share, head hk * share + s % share), so
// that the heads that share keys sit side by side in one workgroup, each key tile is staged once for all of them, and
// the gradients of shared keys are sums inside one workgroup.
//
// Both products run transposed (S^T = K Q^T, O^T = V^T P^T): a lane owns one query (column c of a 16-query block) and
// the accumulators of S^T are, with the K rows of a 32-key group permuted, exactly the B operand of the second product.
// Keys are staged 64 at a time (a wave's lanes are the tile's keys: the mask is one ballot) by LDS-DMA, two tiles in
// turn. Masked keys and rows past the end are fetched from a row of zeros, so that nothing they hold (infinities, NaN)
// reaches a product; their weight is set to exactly 0.
#include "bd_common.h"
#include "bd_prof.h"
#include "bidiff.h"

namespace {

constexpr int KT = 64;         // keys (or query slots) per staged tile
constexpr float LOG2E = 1.44269504088896f;

struct DaArgs {
  const unsigned short *q, *k, *v, *dout;
  const void* lam;
  unsigned short *out, *dq, *dk, *dv;
  float *lse, *maps, *dlam, *stats, *part, *part_ml;
  const unsigned char* mask;
  const int* cu;
  long long qs[3], ks[3], vs[3], ls[3], os[3], dos[3], dqs[3], dks[3], dvs[3], mask_stride;
  int B, Lq, Lk, H, Hkv, share, total, lam_f32, n_blk, n_split;
  float scale;
};

__device__ __attribute__((aligned(64))) const unsigned int bd_da_zero[16] = {};

typedef __attribute__((address_space(3))) void da_lds;

// Byte offset of 16-byte chunk ch of row `row` in a tile of R-byte rows. The XOR spreads what is read at a time over the
// banks: eight rows 0-3 / 8-11 (or 4-7 / 12-15) at one chunk by ds_read_b128, four neighbouring rows of 32 bytes by the
// transposing read.
template <int R>
__device__ __forceinline__ int da_off(int row, int ch) {
  const int f = R >= 256 ? (((row & 3) << 2) | ((row >> 2) & 3))
              : R == 128 ? ((((row >> 1) & 1) << 2) | (((row >> 3) & 1) << 1) | ((row >> 2) & 1))
                         : ((row >> 3) & 3);
  return R * row + 16 * (ch ^ f);
}

__device__ __forceinline__ s16x4 da_read_tr(const unsigned char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}

// 16 (key) x 8 operand of a transposed product: rows r0 .. r0 + 3 and r0 + 4 .. r0 + 7 of the tile, columns 16 dt ..
template <int R>
__device__ __forceinline__ bf16x8 da_frag_tr(const unsigned char* tile, int r0, int dt, int p4) {
  const int ch = 2 * dt + (p4 >> 1);
  union { struct { s16x4 a, b; } s; bf16x8 v; } u;
  u.s.a = da_read_tr(tile + da_off<R>(r0, ch) + 8 * (p4 & 1));
  u.s.b = da_read_tr(tile + da_off<R>(r0 + 4, ch) + 8 * (p4 & 1));
  return u.v;
}

__device__ __forceinline__ void da_dma16(const void* src, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}

// A tile of KT rows of R bytes to LDS in 1-KiB pieces, dealt to NW waves. row_ptr(row) = the row's first byte, or null
// for a row that is to be zeros.
template <int R, int NW, typename F>
__device__ __forceinline__ void da_stage(unsigned lds, int wave, int lane, F row_ptr) {
  constexpr int PIECES = KT * R / 1024, CPR = R / 16;
#pragma unroll
  for (int j = 0; j < (PIECES + NW - 1) / NW; ++j) {
    const int piece = wave + NW * j;
    if (PIECES % NW != 0 && piece >= PIECES) break;
    const int at = piece * 1024 + lane * 16, row = at / R, slot = (at / 16) % CPR;
    const int ch = ((da_off<R>(row, slot) - R * row) >> 4);       // the XOR is its own inverse
    const unsigned char* p = row_ptr(row);
    const unsigned char* src = p ? p + 16 * ch : (const unsigned char*)bd_da_zero;
    da_dma16(src, lds + piece * 1024);
  }
}

struct DaSpan {          // one sequence: first row of queries / keys, their counts, the batch index for strides
  long long q0, k0;
  int Lq, Lk;
};

__device__ __forceinline__ DaSpan da_span(const DaArgs& a, int b) {
  DaSpan s;
  if (a.cu) {            // (offsets are held inside the tensors whatever the table says)
    const int lo = min(max(a.cu[b], 0), a.total), hi = min(max(a.cu[b + 1], lo), a.total);
    s.q0 = s.k0 = lo;
    s.Lq = s.Lk = min(hi - lo, a.Lq);
  } else {
    s.q0 = 0; s.k0 = 0; s.Lq = a.Lq; s.Lk = a.Lk;
  }
  return s;
}

__device__ __forceinline__ float da_lam(const DaArgs& a, long long off) {
  return a.lam_f32 ? ((const float*)a.lam)[off] : bd_bf16_to_f32(((const unsigned short*)a.lam)[off]);
}

// one past the last visible key of the sequence (the tiles behind it are not visited); all threads return it
template <int NT>
__device__ __forceinline__ int da_visible_end(const DaArgs& a, int b, int Lk, int tid, int* red) {
  if (!a.mask) return Lk;
  const unsigned char* m = a.mask + b * a.mask_stride;
  int last = 0;
  for (int j = tid; j < Lk; j += NT) last = m[j] ? j + 1 : last;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o, 64));
  if ((tid & 63) == 0) red[tid >> 6] = last;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) last = max(last, red[w]);
  __syncthreads();
  return last;
}

// mask byte of the lane's key of a tile (0 past the end); a volatile load stays where it is written
__device__ __forceinline__ unsigned da_mask_byte(const DaArgs& a, int b, int key, int end) {
  if (key >= end) return 0u;
  if (!a.mask) return 1u;
  return *(const volatile unsigned char*)(a.mask + b * a.mask_stride + key);
}

// block -> (query block or key block, key head, sequence): each XCD works through one contiguous part of the list, so
// that the blocks of one sequence and head find its rows in their XCD's L2
__device__ __forceinline__ void da_block(int n_blk, int n_heads, int& blk, int& hk, int& b) {
  const int n_all = gridDim.x, xcd = blockIdx.x & 7, q = n_all >> 3, rr = n_all & 7;
  const int lin = (xcd < rr ? xcd * (q + 1) : rr * (q + 1) + (xcd - rr) * q) + (blockIdx.x >> 3);
  blk = lin % n_blk;
  const int t = lin / n_blk;
  hk = t % n_heads;
  b = t / n_heads;
}

// packed rows that belong to no sequence (behind cu[B]): zeros, heads hk * share .. of width W
__device__ __forceinline__ void da_zero_tail(unsigned short* p, const long long* st, int first, int end, int head0, int heads,
                                             int W, int tid, int nt) {
  const int per = heads * (W / 8);
  for (long long i = tid; i < (long long)(end - first) * per; i += nt) {
    const int row = first + (int)(i / per), r = (int)(i % per);
    *(u32x4*)(p + row * st[1] + (long long)(head0 + r / (W / 8)) * st[2] + 8 * (r % (W / 8))) = (u32x4){0u, 0u, 0u, 0u};
  }
}

// =====================================================================================
// Forward. Waves work in pairs: wave 2 w + m holds map m of the 16 QB slots of query group w (NQG groups in a
// workgroup). Split over keys (n_split > 1): each split leaves its unnormalised sums, maximum and normaliser.
// =====================================================================================
template <int D, int QB, int NQG>
__global__ __launch_bounds__(128 * NQG, 2) void da_fwd_kernel(DaArgs a) {
  constexpr int E = 2 * D, KS = D / 32, DT = E / 16, NW = 2 * NQG, RK = 2 * D, RV = 2 * E;
  constexpr int TILE = KT * (2 * RK + RV), SLOTS = 16 * QB * NQG;
  extern __shared__ __attribute__((aligned(1024))) unsigned char da_smem[];
  __shared__ int red[NW];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int map = wave & 1, grp = wave >> 1;
  const int g = lane >> 4, c = lane & 15, q4 = c >> 2, p4 = c & 3;
  int blk, hk, b;
  da_block(a.n_blk * a.n_split, a.Hkv, blk, hk, b);
  const int split = blk % a.n_split;
  blk /= a.n_split;
  if (a.cu && b == a.B) {                                  // (packed: one more sequence, the rows behind the last one)
    if (blk == 0) {
      da_zero_tail(a.out, a.os, min(max(a.cu[a.B], 0), a.total), a.total, hk * a.share, a.share, E, tid, 64 * NW);
      for (int i = 0; i < a.B; ++i) {                      // a sequence longer than Lq: its rows past Lq are NaN, not silence
        const int lo = min(max(a.cu[i], 0), a.total), hi = min(max(a.cu[i + 1], lo), a.total);
        for (long long r = lo + (long long)a.Lq; r < hi; ++r)
          for (int e = tid; e < a.share * E; e += 64 * NW)
            a.out[r * a.os[1] + (long long)(hk * a.share + e / E) * a.os[2] + e % E] = 0x7fc0;
      }
    }
    return;
  }
  const DaSpan sp = da_span(a, b);
  const int n_slots = sp.Lq * a.share;
  if (blk * SLOTS >= n_slots) return;
  const long long bq = a.cu ? 0 : b;                       // batch index of the strided operands

  int kend = da_visible_end<64 * NW>(a, b, sp.Lk, tid, red);
  int kbeg = 0;
  if (a.n_split > 1) {                                     // this split's whole tiles
    const int tiles = (kend + KT - 1) / KT, per = (tiles + a.n_split - 1) / a.n_split;
    kbeg = min(split * per * KT, kend);
    kend = min((split + 1) * per * KT, kend);
  }

  // the lane's slots (column c of each block) and their query fragments
  const int s0 = blk * SLOTS + grp * 16 * QB;
  int row[QB], head[QB];
  bool ok[QB];
  bf16x8 qf[QB][KS];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    int s = s0 + 16 * qb + c;
    ok[qb] = s < n_slots;
    s = ok[qb] ? s : n_slots - 1;
    row[qb] = s / a.share;
    head[qb] = hk * a.share + (s - row[qb] * a.share);
    const unsigned short* qp = a.q + bq * a.qs[0] + (sp.q0 + row[qb]) * a.qs[1] + (2 * head[qb] + map) * a.qs[2] + 8 * g;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[qb][ks] = *(const bf16x8*)(qp + 32 * ks);
  }
  f32x4 o[QB][DT];
  float m_run[QB], l_run[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    m_run[qb] = -INFINITY; l_run[qb] = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[qb][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  const float scale2 = a.scale * LOG2E;

  const unsigned char* const kb0 = (const unsigned char*)(a.k + bq * a.ks[0] + sp.k0 * a.ks[1] + (long long)(2 * hk) * a.ks[2]);
  const unsigned char* const kb1 = kb0 + 2 * a.ks[2];
  const unsigned char* const vb = (const unsigned char*)(a.v + bq * a.vs[0] + sp.k0 * a.vs[1] + (long long)hk * a.vs[2]);
  const unsigned lds0 = (unsigned)(size_t)(da_lds*)da_smem;
  auto stage = [&](int kt0, unsigned long long vis, int buf) {
    const unsigned base = lds0 + buf * TILE;
    auto at = [&](const unsigned char* p, long long st) {
      return [=](int r) { return ((vis >> r) & 1ull) ? p + 2 * st * (kt0 + r) : (const unsigned char*)nullptr; };
    };
    da_stage<RK, NW>(base, wave, lane, at(kb0, a.ks[1]));
    da_stage<RK, NW>(base + KT * RK, wave, lane, at(kb1, a.ks[1]));
    da_stage<RV, NW>(base + 2 * KT * RK, wave, lane, at(vb, a.vs[1]));
  };
  unsigned mb = da_mask_byte(a, b, kbeg + lane, kend);
  unsigned long long vis = __ballot(mb != 0u);
  if (kbeg < kend) stage(kbeg, vis, 0);
  mb = da_mask_byte(a, b, kbeg + KT + lane, kend);
  int buf = 0;
  for (int kt0 = kbeg; kt0 < kend; kt0 += KT, buf ^= 1) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // this tile is there, nobody reads the other buffer
    const unsigned long long vis_next = __ballot(mb != 0u);
    mb = da_mask_byte(a, b, kt0 + 2 * KT + lane, kend);
    if (kt0 + KT < kend) stage(kt0 + KT, vis_next, buf ^ 1);
    const unsigned char* const Ks = da_smem + buf * TILE + map * KT * RK;
    const unsigned char* const Vs = da_smem + buf * TILE + 2 * KT * RK;

    // S^T: s[qb][t][r] <-> key 32 (t >> 1) + 8 g + 4 (t & 1) + r of the tile, slot c of block qb
    f32x4 s[QB][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int krow = 32 * (t >> 1) + 8 * q4 + 4 * (t & 1) + p4;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) s[qb][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16x8 kf = *(const bf16x8*)(Ks + da_off<RK>(krow, 4 * ks + g));
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) s[qb][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[qb][ks], s[qb][t], 0, 0, 0);
      }
    }
    bf16x8 pf[QB][2];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      if (vis != ~0ull) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const unsigned m4 = (unsigned)(vis >> (32 * (t >> 1) + 8 * g + 4 * (t & 1))) & 0xfu;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!((m4 >> r) & 1u)) s[qb][t][r] = -INFINITY;
        }
      }
      float mloc = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t) mloc = fmaxf(fmaxf(mloc, fmaxf(s[qb][t][0], s[qb][t][1])), fmaxf(s[qb][t][2], s[qb][t][3]));
      mloc = fmaxf(mloc, __shfl_xor(mloc, 16, 64));
      mloc = fmaxf(mloc, __shfl_xor(mloc, 32, 64));
      if (__any(mloc > m_run[qb])) {                       // some slot's maximum rises: rescale what was summed
        const float m_new = fmaxf(m_run[qb], mloc);
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_run[qb] - m_new) * scale2);
        l_run[qb] *= alpha;
        m_run[qb] = m_new;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[qb][i][r] *= alpha;
      }
      const float msc = (m_run[qb] == -INFINITY ? 0.f : m_run[qb]) * scale2;     // no visible key so far: every weight 2^-inf = 0
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(s[qb][t][r] * scale2 - msc);
          l_run[qb] += p;                                  // the lane's own keys; the four lanes of a slot are added up at the end
          // weights to bf16 for the second product (half a step: 2^-9 of each weight; the normaliser keeps them in fp32)
          pf[qb][t >> 1][4 * (t & 1) + r] = (__bf16)p;
        }
    }
    // O^T += V^T P^T
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        const bf16x8 vf = da_frag_tr<RV>(Vs, 32 * h2 + 8 * g + q4, dt, p4);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) o[qb][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[qb][h2], o[qb][dt], 0, 0, 0);
      }
    vis = vis_next;
  }
  // lane holds O[slot c of block qb][16 dt + 4 g + r] of its map
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    l_run[qb] += __shfl_xor(l_run[qb], 16, 64);
    l_run[qb] += __shfl_xor(l_run[qb], 32, 64);
  }
  if (a.n_split > 1) {
    const long long pb = ((long long)(b * a.Hkv + hk) * a.n_blk + blk) * a.n_split + split;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const long long at = (pb * 2 + map) * SLOTS + grp * 16 * QB + 16 * qb + c;
      if (ok[qb]) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *(f32x4*)(a.part + at * E + 16 * dt + 4 * g) = o[qb][dt];
        if (g == 0) *(f32x2*)(a.part_ml + 2 * at) = (f32x2){m_run[qb] * scale2, l_run[qb]};
      }
    }
    return;
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float inv = l_run[qb] > 0.f || l_run[qb] != l_run[qb] ? 1.0f / l_run[qb] : 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[qb][dt][r] *= inv;
    const long long rh = (bq * a.Lq + sp.q0 + row[qb]) * a.H + head[qb];       // row and head, counted through the batch
    if (ok[qb] && a.lse && g == 0)         // base 2, for the scaled scores; +inf: no visible key, every weight 2^-inf = 0
      a.lse[2 * rh + map] = l_run[qb] > 0.f || l_run[qb] != l_run[qb] ? m_run[qb] * scale2 + __log2f(l_run[qb]) : INFINITY;
    if (ok[qb] && a.maps) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *(f32x4*)(a.maps + (2 * rh + map) * E + 16 * dt + 4 * g) = o[qb][dt];
    }
  }
  // map 1's sums go to their partner wave through LDS (same lane layout), which joins and stores
  __syncthreads();
  f32x4* const xch = (f32x4*)(da_smem + grp * QB * DT * 1024);
  if (map == 1) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) xch[(qb * DT + dt) * 64 + lane] = o[qb][dt];
  }
  __syncthreads();
  if (map == 0) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      if (!ok[qb]) continue;
      const float lam = da_lam(a, bq * a.ls[0] + (sp.q0 + row[qb]) * a.ls[1] + head[qb] * a.ls[2]);
      unsigned short* op = a.out + bq * a.os[0] + (sp.q0 + row[qb]) * a.os[1] + head[qb] * a.os[2] + 4 * g;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const f32x4 o2 = xch[(qb * DT + dt) * 64 + lane];
        u32x2 w;
        w[0] = bd_pack_bf16x2(o[qb][dt][0] - lam * o2[0], o[qb][dt][1] - lam * o2[1]);
        w[1] = bd_pack_bf16x2(o[qb][dt][2] - lam * o2[2], o[qb][dt][3] - lam * o2[3]);
        *(u32x2*)(op + 16 * dt) = w;
      }
    }
  }
}

// joins the key splits of one slot: a workgroup of E threads, thread = value column
template <int D, int SLOTS>
__global__ __launch_bounds__(2 * D) void da_join_kernel(DaArgs a) {
  constexpr int E = 2 * D;
  const int e = threadIdx.x;
  const int slot = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int blk = slot / SLOTS, in_blk = slot - blk * SLOTS;
  const int row = slot / a.share, head = hk * a.share + (slot - row * a.share);
  float r[2];
  const long long rh = ((long long)b * a.Lq + row) * a.H + head;
#pragma unroll
  for (int map = 0; map < 2; ++map) {
    const long long at0 = (((long long)(b * a.Hkv + hk) * a.n_blk + blk) * a.n_split * 2 + map) * SLOTS + in_blk;
    float m = -INFINITY;
    for (int i = 0; i < a.n_split; ++i) m = fmaxf(m, a.part_ml[2 * (at0 + (long long)i * 2 * SLOTS)]);
    float l = 0.f, o = 0.f;
    for (int i = 0; i < a.n_split; ++i) {
      const long long at = at0 + (long long)i * 2 * SLOTS;
      const float li = a.part_ml[2 * at + 1];
      if (li == 0.f) continue;                             // a split without a visible key
      const float w = __builtin_amdgcn_exp2f(a.part_ml[2 * at] - m);
      l += w * li;
      o += w * a.part[at * E + e];
    }
    const bool any = l > 0.f || l != l;
    r[map] = any ? o / l : 0.f;
    if (a.lse && e == 0) a.lse[2 * rh + map] = any ? m + __log2f(l) : INFINITY;
    if (a.maps) a.maps[(2 * rh + map) * E + e] = r[map];
  }
  const float lam = da_lam(a, b * a.ls[0] + row * a.ls[1] + head * a.ls[2]);
  a.out[b * a.os[0] + row * a.os[1] + head * a.os[2] + e] = bd_f32_to_bf16(r[0] - lam * r[1]);
}

// =====================================================================================
// Backward, query side: dQ and what the key side needs of each slot (stats: lse1, lse2, delta1, delta2, lam), dlam.
// A wave owns 16 QB slots and both of their maps (dP = dO V^T is shared). delta_m comes from the forward's fp32 maps
// (dO . O_m) or, where none were kept, from a first walk over the keys: sums of the very P and dP that form dS.
// From a bf16-rounded O it would miss sum_j dS_ij = 0 by 2^-9 of |dO||O| for all keys alike, as large as dS itself
// where attention is nearly uniform.
// =====================================================================================
template <int D, int QB>
__global__ __launch_bounds__(256, 1) void da_bwd_dq_kernel(DaArgs a) {
  constexpr int E = 2 * D, KS = D / 32, ES = E / 32, DT = D / 16, NW = 4, RK = 2 * D, RV = 2 * E;
  constexpr int TILE = KT * (2 * RK + RV), SLOTS = 64 * QB;
  extern __shared__ __attribute__((aligned(1024))) unsigned char da_smem[];
  __shared__ int red[NW];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15, q4 = c >> 2, p4 = c & 3;
  int blk, hk, b;
  da_block(a.n_blk, a.Hkv, blk, hk, b);
  if (a.cu && b == a.B) {
    if (blk == 0) {
      const int first = min(max(a.cu[a.B], 0), a.total);
      da_zero_tail(a.dq, a.dqs, first, a.total, 2 * hk * a.share, 2 * a.share, D, tid, 256);
      for (long long i = tid; i < (long long)(a.total - first) * a.share; i += 256)
        a.dlam[(first + i / a.share) * a.H + hk * a.share + i % a.share] = 0.f;
    }
    return;
  }
  const DaSpan sp = da_span(a, b);
  const int n_slots = sp.Lq * a.share;
  if (blk * SLOTS >= n_slots) return;
  const long long bq = a.cu ? 0 : b;
  const int kend = da_visible_end<256>(a, b, sp.Lk, tid, red);

  const int s0 = blk * SLOTS + wave * 16 * QB;
  int row[QB], head[QB];
  bool ok[QB];
  long long rh[QB];
  bf16x8 qf[QB][2][KS], dof[QB][ES];
  float lse[QB][2], dl[QB][2];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    int s = s0 + 16 * qb + c;
    ok[qb] = s < n_slots;
    s = ok[qb] ? s : n_slots - 1;
    row[qb] = s / a.share;
    head[qb] = hk * a.share + (s - row[qb] * a.share);
    rh[qb] = (bq * a.Lq + sp.q0 + row[qb]) * a.H + head[qb];
    const unsigned short* dp = a.dout + bq * a.dos[0] + (sp.q0 + row[qb]) * a.dos[1] + head[qb] * a.dos[2] + 8 * g;
#pragma unroll
    for (int ks = 0; ks < ES; ++ks) dof[qb][ks] = *(const bf16x8*)(dp + 32 * ks);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const unsigned short* qp = a.q + bq * a.qs[0] + (sp.q0 + row[qb]) * a.qs[1] + (2 * head[qb] + m) * a.qs[2] + 8 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[qb][m][ks] = *(const bf16x8*)(qp + 32 * ks);
      lse[qb][m] = a.lse[2 * rh[qb] + m];
      dl[qb][m] = 0.f;
      if (a.maps) {
        const float* op = a.maps + (2 * rh[qb] + m) * E + 8 * g;
#pragma unroll
        for (int ks = 0; ks < ES; ++ks) {
          const f32x4 x = *(const f32x4*)(op + 32 * ks), y = *(const f32x4*)(op + 32 * ks + 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) dl[qb][m] += (float)dof[qb][ks][r] * x[r] + (float)dof[qb][ks][4 + r] * y[r];
        }
        dl[qb][m] += __shfl_xor(dl[qb][m], 16, 64);
        dl[qb][m] += __shfl_xor(dl[qb][m], 32, 64);
      }
    }
  }
  f32x4 acc[QB][2][DT];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[qb][m][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const float scale2 = a.scale * LOG2E;

  const unsigned char* const kb0 = (const unsigned char*)(a.k + bq * a.ks[0] + sp.k0 * a.ks[1] + (long long)(2 * hk) * a.ks[2]);
  const unsigned char* const kb1 = kb0 + 2 * a.ks[2];
  const unsigned char* const vb = (const unsigned char*)(a.v + bq * a.vs[0] + sp.k0 * a.vs[1] + (long long)hk * a.vs[2]);
  const unsigned lds0 = (unsigned)(size_t)(da_lds*)da_smem;
  auto stage = [&](int kt0, unsigned long long vis, int buf) {
    const unsigned base = lds0 + buf * TILE;
    auto at = [&](const unsigned char* p, long long st) {
      return [=](int r) { return ((vis >> r) & 1ull) ? p + 2 * st * (kt0 + r) : (const unsigned char*)nullptr; };
    };
    da_stage<RK, NW>(base, wave, lane, at(kb0, a.ks[1]));
    da_stage<RK, NW>(base + KT * RK, wave, lane, at(kb1, a.ks[1]));
    da_stage<RV, NW>(base + 2 * KT * RK, wave, lane, at(vb, a.vs[1]));
  };
  for (int walk = a.maps ? 1 : 0; walk < 2; ++walk) {
    unsigned mb = da_mask_byte(a, b, lane, kend);
    unsigned long long vis = __ballot(mb != 0u);
    __syncthreads();                                       // (second walk: nobody reads the first one's last tile)
    if (kend > 0) stage(0, vis, 0);
    mb = da_mask_byte(a, b, KT + lane, kend);
    int buf = 0;
    for (int kt0 = 0; kt0 < kend; kt0 += KT, buf ^= 1) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const unsigned long long vis_next = __ballot(mb != 0u);
      mb = da_mask_byte(a, b, kt0 + 2 * KT + lane, kend);
      if (kt0 + KT < kend) stage(kt0 + KT, vis_next, buf ^ 1);
      const unsigned char* const K0 = da_smem + buf * TILE;
      const unsigned char* const K1 = K0 + KT * RK;
      const unsigned char* const Vs = K0 + 2 * KT * RK;
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {                     // 32 keys
        bf16x8 dsf[QB][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int krow = 32 * h2 + 8 * q4 + 4 * half + p4;
          f32x4 s[QB][2], dp[QB];
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) s[qb][0] = s[qb][1] = dp[qb] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const bf16x8 k0f = *(const bf16x8*)(K0 + da_off<RK>(krow, 4 * ks + g));
            const bf16x8 k1f = *(const bf16x8*)(K1 + da_off<RK>(krow, 4 * ks + g));
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
              s[qb][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0f, qf[qb][0][ks], s[qb][0], 0, 0, 0);
              s[qb][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1f, qf[qb][1][ks], s[qb][1], 0, 0, 0);
            }
          }
#pragma unroll
          for (int ks = 0; ks < ES; ++ks) {
            const bf16x8 vf = *(const bf16x8*)(Vs + da_off<RV>(krow, 4 * ks + g));
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) dp[qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, dof[qb][ks], dp[qb], 0, 0, 0);
          }
          const unsigned m4 = (unsigned)(vis >> (32 * h2 + 8 * g + 4 * half)) & 0xfu;
#pragma unroll
          for (int qb = 0; qb < QB; ++qb)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float p = ((m4 >> r) & 1u) ? __builtin_amdgcn_exp2f(s[qb][m][r] * scale2 - lse[qb][m]) : 0.f;
                if (walk == 0) dl[qb][m] += p * dp[qb][r];
                else dsf[qb][m][4 * half + r] = (__bf16)(p * (dp[qb][r] - dl[qb][m]));
              }
        }
        if (walk == 1) {                                   // dQ^T += K^T dS^T
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const bf16x8 k0t = da_frag_tr<RK>(K0, 32 * h2 + 8 * g + q4, dt, p4);
            const bf16x8 k1t = da_frag_tr<RK>(K1, 32 * h2 + 8 * g + q4, dt, p4);
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
              acc[qb][0][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0t, dsf[qb][0], acc[qb][0][dt], 0, 0, 0);
              acc[qb][1][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1t, dsf[qb][1], acc[qb][1][dt], 0, 0, 0);
            }
          }
        }
      }
      vis = vis_next;
    }
    if (walk == 0) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          dl[qb][m] += __shfl_xor(dl[qb][m], 16, 64);
          dl[qb][m] += __shfl_xor(dl[qb][m], 32, 64);
        }
    }
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    if (!ok[qb]) continue;
    const float lam = da_lam(a, bq * a.ls[0] + (sp.q0 + row[qb]) * a.ls[1] + head[qb] * a.ls[2]);
    if (g == 0) {
      *(f32x4*)(a.stats + 8 * rh[qb]) = (f32x4){lse[qb][0], lse[qb][1], dl[qb][0], dl[qb][1]};
      a.stats[8 * rh[qb] + 4] = lam;
      a.dlam[rh[qb]] = -dl[qb][1];
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const float f = m ? -lam * a.scale : a.scale;
      unsigned short* op = a.dq + bq * a.dqs[0] + (sp.q0 + row[qb]) * a.dqs[1] + (2 * head[qb] + m) * a.dqs[2] + 4 * g;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        u32x2 w;
        w[0] = bd_pack_bf16x2(acc[qb][m][dt][0] * f, acc[qb][m][dt][1] * f);
        w[1] = bd_pack_bf16x2(acc[qb][m][dt][2] * f, acc[qb][m][dt][3] * f);
        *(u32x2*)(op + 16 * dt) = w;
      }
    }
  }
}

// =====================================================================================
// Backward, key side: a workgroup owns 64 KB keys of one key head and walks the query slots of all heads that share it.
// =====================================================================================
template <int D, int KB>
__global__ __launch_bounds__(256, 1) void da_bwd_dkv_kernel(DaArgs a) {
  constexpr int E = 2 * D, KS = D / 32, ES = E / 32, DT = D / 16, ET = E / 16, NW = 4, RK = 2 * D, RV = 2 * E;
  constexpr int TILE = KT * (2 * RK + RV + 32), KEYS = 64 * KB;
  extern __shared__ __attribute__((aligned(1024))) unsigned char da_smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15, q4 = c >> 2, p4 = c & 3;
  int blk, hk, b;
  da_block(a.n_blk, a.Hkv, blk, hk, b);
  if (a.cu && b == a.B) {
    if (blk == 0) {
      const int first = min(max(a.cu[a.B], 0), a.total);
      da_zero_tail(a.dk, a.dks, first, a.total, 2 * hk, 2, D, tid, 256);
      da_zero_tail(a.dv, a.dvs, first, a.total, hk, 1, E, tid, 256);
    }
    return;
  }
  const DaSpan sp = da_span(a, b);
  if (blk * KEYS >= sp.Lk) return;
  const long long bq = a.cu ? 0 : b;
  const int n_slots = sp.Lq * a.share;
  const int k0 = blk * KEYS + wave * 16 * KB;
  bool inside[KB], vis[KB];
  bool live = false;
  bf16x8 kf[KB][2][KS], vf[KB][ES];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    int key = k0 + 16 * kb + c;
    inside[kb] = key < sp.Lk;
    key = inside[kb] ? key : sp.Lk - 1;
    vis[kb] = inside[kb] && (!a.mask || a.mask[b * a.mask_stride + key] != 0);
    live = live || vis[kb];
    const unsigned short* vp = a.v + bq * a.vs[0] + (sp.k0 + key) * a.vs[1] + hk * a.vs[2] + 8 * g;
#pragma unroll
    for (int ks = 0; ks < ES; ++ks) vf[kb][ks] = *(const bf16x8*)(vp + 32 * ks);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const unsigned short* kp = a.k + bq * a.ks[0] + (sp.k0 + key) * a.ks[1] + (2 * hk + m) * a.ks[2] + 8 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[kb][m][ks] = *(const bf16x8*)(kp + 32 * ks);
    }
  }
  f32x4 ak[KB][2][DT], av[KB][ET];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
    for (int i = 0; i < DT; ++i) ak[kb][0][i] = ak[kb][1][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < ET; ++i) av[kb][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  const float scale2 = a.scale * LOG2E;
  const unsigned lds0 = (unsigned)(size_t)(da_lds*)da_smem;
  auto stage = [&](int t0, int buf) {
    const unsigned base = lds0 + buf * TILE;
    auto at = [&](const unsigned short* p, const long long* st, int mul, int add) {
      return [=](int r) {
        const int s = t0 + r;
        if (s >= n_slots) return (const unsigned char*)nullptr;
        const int row = s / a.share, head = hk * a.share + (s - row * a.share);
        return (const unsigned char*)(p + bq * st[0] + (sp.q0 + row) * st[1] + (mul * head + add) * st[2]);
      };
    };
    da_stage<RK, NW>(base, wave, lane, at(a.q, a.qs, 2, 0));
    da_stage<RK, NW>(base + KT * RK, wave, lane, at(a.q, a.qs, 2, 1));
    da_stage<RV, NW>(base + 2 * KT * RK, wave, lane, at(a.dout, a.dos, 1, 0));
    if (wave < 2) {                                        // the slots' statistics: lane = slot, 16 bytes a wave
      const int s = t0 + lane;
      const unsigned char* src = (const unsigned char*)bd_da_zero;
      if (s < n_slots) {
        const int row = s / a.share, head = hk * a.share + (s - row * a.share);
        src = (const unsigned char*)(a.stats + 8 * ((bq * a.Lq + sp.q0 + row) * a.H + head) + 4 * wave);
      }
      da_dma16(src, base + KT * (2 * RK + RV) + wave * 1024);
    }
  };
  if (__syncthreads_or(live)) {                            // no visible key in this workgroup: every gradient is zero
    stage(0, 0);
    int buf = 0;
    for (int t0 = 0; t0 < n_slots; t0 += KT, buf ^= 1) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (t0 + KT < n_slots) stage(t0 + KT, buf ^ 1);
      const unsigned char* const Q0 = da_smem + buf * TILE;
      const unsigned char* const Q1 = Q0 + KT * RK;
      const unsigned char* const Ds = Q0 + 2 * KT * RK;
      const f32x4* const St = (const f32x4*)(Ds + KT * RV);        // [64] lse1, lse2, delta1, delta2; then [64] lam, ...
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {                     // 32 slots
        bf16x8 pf[KB], dsf[KB][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int srow = 32 * h2 + 8 * q4 + 4 * half + p4;
          f32x4 s[KB][2], dp[KB];
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) s[kb][0] = s[kb][1] = dp[kb] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const bf16x8 q0f = *(const bf16x8*)(Q0 + da_off<RK>(srow, 4 * ks + g));
            const bf16x8 q1f = *(const bf16x8*)(Q1 + da_off<RK>(srow, 4 * ks + g));
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              s[kb][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q0f, kf[kb][0][ks], s[kb][0], 0, 0, 0);
              s[kb][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q1f, kf[kb][1][ks], s[kb][1], 0, 0, 0);
            }
          }
#pragma unroll
          for (int ks = 0; ks < ES; ++ks) {
            const bf16x8 df = *(const bf16x8*)(Ds + da_off<RV>(srow, 4 * ks + g));
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) dp[kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(df, vf[kb][ks], dp[kb], 0, 0, 0);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int sl = 32 * h2 + 8 * g + 4 * half + r;
            const f32x4 st = St[sl];
            const float lam = *(const float*)(St + KT + sl);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              const float p1 = __builtin_amdgcn_exp2f(s[kb][0][r] * scale2 - st[0]);
              const float p2 = __builtin_amdgcn_exp2f(s[kb][1][r] * scale2 - st[1]) * lam;
              pf[kb][4 * half + r] = (__bf16)(p1 - p2);
              dsf[kb][0][4 * half + r] = (__bf16)(p1 * (dp[kb][r] - st[2]));
              dsf[kb][1][4 * half + r] = (__bf16)(p2 * (st[3] - dp[kb][r]));
            }
          }
        }
#pragma unroll
        for (int dt = 0; dt < ET; ++dt) {
          const bf16x8 dt_ = da_frag_tr<RV>(Ds, 32 * h2 + 8 * g + q4, dt, p4);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) av[kb][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(dt_, pf[kb], av[kb][dt], 0, 0, 0);
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const bf16x8 q0t = da_frag_tr<RK>(Q0, 32 * h2 + 8 * g + q4, dt, p4);
          const bf16x8 q1t = da_frag_tr<RK>(Q1, 32 * h2 + 8 * g + q4, dt, p4);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            ak[kb][0][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q0t, dsf[kb][0], ak[kb][0][dt], 0, 0, 0);
            ak[kb][1][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q1t, dsf[kb][1], ak[kb][1][dt], 0, 0, 0);
          }
        }
      }
    }
  }
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    if (!inside[kb]) continue;
    const int key = k0 + 16 * kb + c;
    // a masked key's gradients are exact zeros whatever its column held
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      unsigned short* op = a.dk + bq * a.dks[0] + (sp.k0 + key) * a.dks[1] + (2 * hk + m) * a.dks[2] + 4 * g;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        u32x2 w = {0u, 0u};
        if (vis[kb]) {
          w[0] = bd_pack_bf16x2(ak[kb][m][dt][0] * a.scale, ak[kb][m][dt][1] * a.scale);
          w[1] = bd_pack_bf16x2(ak[kb][m][dt][2] * a.scale, ak[kb][m][dt][3] * a.scale);
        }
        *(u32x2*)(op + 16 * dt) = w;
      }
    }
    unsigned short* op = a.dv + bq * a.dvs[0] + (sp.k0 + key) * a.dvs[1] + hk * a.dvs[2] + 4 * g;
#pragma unroll
    for (int dt = 0; dt < ET; ++dt) {
      u32x2 w = {0u, 0u};
      if (vis[kb]) {
        w[0] = bd_pack_bf16x2(av[kb][dt][0], av[kb][dt][1]);
        w[1] = bd_pack_bf16x2(av[kb][dt][2], av[kb][dt][3]);
      }
      *(u32x2*)(op + 16 * dt) = w;
    }
  }
}

// dlam [B, L, H] summed over the axes that lam was broadcast along (kept axes: kb, kl, kh), in a fixed order; one
// workgroup per kept value (a wave's worth of values per workgroup where nothing is summed: a cast)
template <typename T>
__global__ __launch_bounds__(256) void da_dlam_kernel(const float* __restrict__ dlam, T* __restrict__ out, int B, int L, int H, int kb, int kl,
                                                      int kh) {
  __shared__ float part[4];
  const int nh = kh ? H : 1, nl = kl ? L : 1;
  const int h = blockIdx.x % nh, l = (blockIdx.x / nh) % nl, b = blockIdx.x / nh / nl;
  const int sb = kb ? 1 : B, sl = kl ? 1 : L, sh = kh ? 1 : H;
  const long long n = (long long)sb * sl * sh;
  float s = 0.f;
  for (long long i = threadIdx.x; i < n; i += 256) {
    const int ih = (int)(i % sh), il = (int)(i / sh % sl), ib = (int)(i / sh / sl);
    s += dlam[((long long)(b + ib) * L + l + il) * H + h + ih];
  }
  s = bd_wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = (part[0] + part[1]) + (part[2] + part[3]);
    if (sizeof(T) == 2) out[blockIdx.x] = (T)bd_f32_to_bf16(s);
    else ((float*)out)[blockIdx.x] = s;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void da_dlam_cast_kernel(const float* __restrict__ dlam, T* __restrict__ out, long long n) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  if (sizeof(T) == 2) out[i] = (T)bd_f32_to_bf16(dlam[i]);
  else ((float*)out)[i] = dlam[i];
}

// ---------------------------------------------------------------------------------------------- host side
constexpr int FWD_QB = 2, FWD_NQG = 4, FWD_SLOTS = 16 * FWD_QB * FWD_NQG;      // 128 slots, 8 waves
constexpr int ROWS_NQG = 2, ROWS_SLOTS = 16 * ROWS_NQG;                         // few slots: 32, 4 waves of 16

int da_splits(const bd_diff_attn_args& p) {
  // few slots against many keys: enough splits of whole key tiles for two workgroups per CU, four tiles each at least
  if (p.cu_seqlens) return 1;
  const long long slots = (long long)p.Lq * (p.H / p.Hkv);
  if (slots > FWD_SLOTS) return 1;
  const long long blocks = (long long)p.B * p.Hkv * ((slots + ROWS_SLOTS - 1) / ROWS_SLOTS);
  const int tiles = (p.Lk + KT - 1) / KT;
  long long n = 512 / (blocks > 0 ? blocks : 1);
  if (n > tiles / 4) n = tiles / 4;
  return n < 1 ? 1 : n > 256 ? 256 : (int)n;
}

bool da_few(const bd_diff_attn_args& p) { return (long long)p.Lq * (p.H / p.Hkv) <= ROWS_SLOTS || da_splits(p) > 1; }

int da_check(const bd_diff_attn_args& p, const char* what, DaArgs& a) {
  BD_REQUIRE(p.q && p.k && p.v && p.lam, "%s: null operand", what);
  BD_REQUIRE(p.B > 0 && p.Lq > 0 && p.Lk > 0 && p.H > 0 && p.Hkv > 0, "%s: empty shape", what);
  BD_REQUIRE(p.H % p.Hkv == 0, "%s: %d heads cannot share %d key heads evenly", what, p.H, p.Hkv);
  BD_REQUIRE(p.head_dim == 32 || p.head_dim == 64 || p.head_dim == 128, "%s: head_dim %d not in {32, 64, 128}", what, p.head_dim);
  BD_REQUIRE((long long)p.Lq * (p.H / p.Hkv) < (1ll << 30) && p.Lk < (1 << 30) && (long long)p.B * p.Hkv < (1ll << 24),
             "%s: too many rows or heads", what);
  BD_REQUIRE(!p.cu_seqlens || p.Lq == p.Lk, "%s: packed rows need Lq == Lk (the longest sequence)", what);
  BD_REQUIRE(!p.cu_seqlens || p.total_rows > 0, "%s: packed rows need total_rows", what);
  BD_REQUIRE(p.scale > 0.f, "%s: scale must be positive", what);
  BD_REQUIRE(p.lam_dtype == BD_DTYPE_BF16 || p.lam_dtype == BD_DTYPE_F32, "%s: lam is neither bf16 nor fp32", what);
  const void* aligned[] = {p.q, p.k, p.v};
  for (const void* x : aligned) BD_REQUIRE(((uintptr_t)x & 15) == 0, "%s: q, k and v must be 16-byte aligned", what);
  for (int i = 0; i < 3; ++i)
    BD_REQUIRE(p.q_stride[i] % 8 == 0 && p.k_stride[i] % 8 == 0 && p.v_stride[i] % 8 == 0,
               "%s: q, k and v strides must be multiples of 8 elements", what);
  a = DaArgs();
  a.q = (const unsigned short*)p.q; a.k = (const unsigned short*)p.k; a.v = (const unsigned short*)p.v; a.lam = p.lam;
  a.mask = p.key_mask; a.cu = p.cu_seqlens; a.mask_stride = p.key_mask_stride;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = p.q_stride[i]; a.ks[i] = p.k_stride[i]; a.vs[i] = p.v_stride[i]; a.ls[i] = p.lam_stride[i]; a.os[i] = p.out_stride[i];
    a.dos[i] = p.dout_stride[i]; a.dqs[i] = p.dq_stride[i]; a.dks[i] = p.dk_stride[i]; a.dvs[i] = p.dv_stride[i];
  }
  a.B = p.B; a.Lq = p.Lq; a.Lk = p.Lk; a.H = p.H; a.Hkv = p.Hkv; a.share = p.H / p.Hkv; a.total = p.total_rows;
  a.lam_f32 = p.lam_dtype == BD_DTYPE_F32; a.scale = p.scale; a.n_split = 1;
  a.lse = p.lse; a.maps = p.maps;
  return BD_OK;
}

template <int D>
int da_forward(const bd_diff_attn_args& p, DaArgs& a, hipStream_t s) {
  constexpr int LDS = 2 * KT * 8 * D;
  const long long slots = (long long)a.Lq * a.share;
  const int seqs = a.B + (a.cu ? 1 : 0);
  a.n_split = da_splits(p);
  const bool few = da_few(p);
  const int per = few ? ROWS_SLOTS : FWD_SLOTS;
  a.n_blk = (int)((slots + per - 1) / per);
  const long long grid = (long long)a.n_blk * a.n_split * a.Hkv * seqs;
  BD_REQUIRE(grid < (1ll << 31), "bd_diff_attention_fwd: too many workgroups");
  if (a.n_split > 1) {
    const long long ml = (long long)a.n_blk * a.n_split * a.Hkv * a.B * 2 * ROWS_SLOTS;
    a.part_ml = (float*)p.workspace;
    a.part = a.part_ml + ml * 2;
  }
  if (few) {
    BD_SET_MAX_LDS((da_fwd_kernel<D, 1, ROWS_NQG>), LDS);
    hipLaunchKernelGGL((da_fwd_kernel<D, 1, ROWS_NQG>), dim3((unsigned)grid), dim3(128 * ROWS_NQG), LDS, s, a);
    if (a.n_split > 1)
      hipLaunchKernelGGL((da_join_kernel<D, ROWS_SLOTS>), dim3((unsigned)slots, a.Hkv, a.B), dim3(2 * D), 0, s, a);
  } else {
    BD_SET_MAX_LDS((da_fwd_kernel<D, FWD_QB, FWD_NQG>), LDS);
    hipLaunchKernelGGL((da_fwd_kernel<D, FWD_QB, FWD_NQG>), dim3((unsigned)grid), dim3(128 * FWD_NQG), LDS, s, a);
  }
  return bd_check_launch("bd_diff_attention_fwd");
}

template <int D>
int da_backward(DaArgs& a, hipStream_t s) {
  constexpr int LDS = 2 * KT * 8 * D, LDS_KV = 2 * KT * (8 * D + 32);
  const long long slots = (long long)a.Lq * a.share;
  const int seqs = a.B + (a.cu ? 1 : 0);
  a.n_blk = (int)((slots + 63) / 64);
  long long grid = (long long)a.n_blk * a.Hkv * seqs;
  BD_REQUIRE(grid < (1ll << 31), "bd_diff_attention_bwd: too many workgroups");
  BD_SET_MAX_LDS((da_bwd_dq_kernel<D, 1>), LDS);
  hipLaunchKernelGGL((da_bwd_dq_kernel<D, 1>), dim3((unsigned)grid), dim3(256), LDS, s, a);
  a.n_blk = (a.Lk + 63) / 64;
  grid = (long long)a.n_blk * a.Hkv * seqs;
  BD_REQUIRE(grid < (1ll << 31), "bd_diff_attention_bwd: too many workgroups");
  BD_SET_MAX_LDS((da_bwd_dkv_kernel<D, 1>), LDS_KV);
  hipLaunchKernelGGL((da_bwd_dkv_kernel<D, 1>), dim3((unsigned)grid), dim3(256), LDS_KV, s, a);
  return bd_check_launch("bd_diff_attention_bwd");
}

}  // namespace

extern "C" long long bd_diff_attention_workspace_bytes(const bd_diff_attn_args* p, int backward) {
  if (!p || p->B <= 0 || p->Lq <= 0 || p->Lk <= 0 || p->H <= 0 || p->Hkv <= 0 || p->H % p->Hkv) return -1;
  const long long rows = p->cu_seqlens ? p->total_rows : (long long)p->B * p->Lq;
  if (backward) return rows * p->H * 32;
  const int n = da_splits(*p);
  if (n == 1) return 0;
  const long long slots = (long long)p->Lq * (p->H / p->Hkv), blocks = (slots + ROWS_SLOTS - 1) / ROWS_SLOTS;
  return blocks * n * p->Hkv * p->B * 2 * ROWS_SLOTS * (2 + 2 * (long long)p->head_dim) * 4;
}

extern "C" int bd_diff_attention_fwd(const bd_diff_attn_args* p, void* stream) {
  BD_REQUIRE(p != nullptr, "bd_diff_attention_fwd: null arguments");
  DaArgs a;
  const int rc = da_check(*p, "bd_diff_attention_fwd", a);
  if (rc != BD_OK) return rc;
  BD_REQUIRE(p->out && ((uintptr_t)p->out & 15) == 0, "bd_diff_attention_fwd: out must be a 16-byte aligned tensor");
  for (int i = 0; i < 3; ++i) BD_REQUIRE(p->out_stride[i] % 8 == 0, "bd_diff_attention_fwd: out strides must be multiples of 8 elements");
  BD_REQUIRE(!p->maps || (p->lse && ((uintptr_t)p->maps & 15) == 0), "bd_diff_attention_fwd: maps need lse beside them and 16-byte alignment");
  const long long need = bd_diff_attention_workspace_bytes(p, 0);
  BD_REQUIRE(need == 0 || (p->workspace && p->workspace_bytes >= need && ((uintptr_t)p->workspace & 15) == 0),
             "bd_diff_attention_fwd: the workspace must hold %lld bytes, 16-byte aligned", need);
  a.out = (unsigned short*)p->out;
  bd_prof_scope prof(stream, 12.0 * p->B * p->H * (double)p->Lq * p->Lk * p->head_dim, BD_PROF_ATTN_FWD);
  switch (p->head_dim) {
    case 32: return da_forward<32>(*p, a, (hipStream_t)stream);
    case 64: return da_forward<64>(*p, a, (hipStream_t)stream);
    default: return da_forward<128>(*p, a, (hipStream_t)stream);
  }
}

extern "C" int bd_diff_attention_bwd(const bd_diff_attn_args* p, void* stream) {
  BD_REQUIRE(p != nullptr, "bd_diff_attention_bwd: null arguments");
  DaArgs a;
  const int rc = da_check(*p, "bd_diff_attention_bwd", a);
  if (rc != BD_OK) return rc;
  BD_REQUIRE(p->dout && p->dq && p->dk && p->dv && p->dlam && p->lse, "bd_diff_attention_bwd: null operand");
  const void* aligned[] = {p->dout, p->dq, p->dk, p->dv, p->maps};
  for (const void* x : aligned) BD_REQUIRE(((uintptr_t)x & 15) == 0, "bd_diff_attention_bwd: operands must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    BD_REQUIRE(p->dout_stride[i] % 8 == 0 && p->dq_stride[i] % 8 == 0 && p->dk_stride[i] % 8 == 0 && p->dv_stride[i] % 8 == 0,
               "bd_diff_attention_bwd: strides must be multiples of 8 elements");
  const long long need = bd_diff_attention_workspace_bytes(p, 1);
  BD_REQUIRE(p->workspace && p->workspace_bytes >= need && ((uintptr_t)p->workspace & 15) == 0,
             "bd_diff_attention_bwd: the workspace must hold %lld bytes, 16-byte aligned", need);
  a.dout = (const unsigned short*)p->dout;
  a.dq = (unsigned short*)p->dq; a.dk = (unsigned short*)p->dk; a.dv = (unsigned short*)p->dv;
  a.dlam = p->dlam;
  a.stats = (float*)p->workspace;
  bd_prof_scope prof(stream, 28.0 * p->B * p->H * (double)p->Lq * p->Lk * p->head_dim, BD_PROF_ATTN_BWD);
  switch (p->head_dim) {
    case 32: return da_backward<32>(a, (hipStream_t)stream);
    case 64: return da_backward<64>(a, (hipStream_t)stream);
    default: return da_backward<128>(a, (hipStream_t)stream);
  }
}

extern "C" int bd_diff_attention_dlam(const float* dlam, void* out, int out_dtype, int B, int L, int H, int keep_b, int keep_l, int keep_h,
                                      void* stream) {
  BD_REQUIRE(dlam && out && B > 0 && L > 0 && H > 0, "bd_diff_attention_dlam: null operand or empty shape");
  BD_REQUIRE(out_dtype == BD_DTYPE_BF16 || out_dtype == BD_DTYPE_F32, "bd_diff_attention_dlam: out is neither bf16 nor fp32");
  const long long all = (long long)B * L * H, kept = (keep_b ? B : 1ll) * (keep_l ? L : 1) * (keep_h ? H : 1);
  BD_REQUIRE(all < (1ll << 38) && (kept == all || kept < (1ll << 31)), "bd_diff_attention_dlam: too many values");
  hipStream_t s = (hipStream_t)stream;
  const bool bf = out_dtype == BD_DTYPE_BF16;
  if (kept == all) {
    const dim3 grid((unsigned)((all + 255) / 256));
    if (bf) hipLaunchKernelGGL(da_dlam_cast_kernel<unsigned short>, grid, dim3(256), 0, s, dlam, (unsigned short*)out, all);
    else hipLaunchKernelGGL(da_dlam_cast_kernel<float>, grid, dim3(256), 0, s, dlam, (float*)out, all);
  } else {
    const dim3 grid((unsigned)kept);
    if (bf) hipLaunchKernelGGL(da_dlam_kernel<unsigned short>, grid, dim3(256), 0, s, dlam, (unsigned short*)out, B, L, H, keep_b, keep_l, keep_h);
    else hipLaunchKernelGGL(da_dlam_kernel<float>, grid, dim3(256), 0, s, dlam, (float*)out, B, L, H, keep_b, keep_l, keep_h);
  }
  return bd_check_launch("bd_diff_attention_dlam");
}
