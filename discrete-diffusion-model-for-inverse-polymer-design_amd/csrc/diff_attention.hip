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

#include <type_traits>

namespace {

constexpr int KT = 64;         // keys (or query slots) per staged tile
constexpr float LOG2E = 1.44269504088896f;

struct DaArgs {
  const unsigned short *q, *k, *v, *dout;
  const void* lam;
  unsigned short *out, *dq, *dk, *dv;
  float *lse, *maps, *stats, *part, *part_ml;
  void* dlam;
  const unsigned char* mask;
  const int* cu;
  long long qs[3], ks[3], vs[3], ls[3], os[3], dos[3], dqs[3], dks[3], dvs[3], mask_stride;
  int B, Lq, Lk, H, Hkv, share, total, lam_f32, dlam_bf16, n_blk, n_split;
  int per;                       // split over keys: slots of a workgroup of the forward
  unsigned share_mul, share_log; // s / share = (4 s share_mul >> 32) >> share_log for s < 2^30
  int small_strides;             // 64 rows of every operand lie within 4 GiB: staged by 32-bit offsets
  float scale;
};

// row and head (of those that share a key head) of slot s
__device__ __forceinline__ void da_split(const DaArgs& a, int s, int& row, int& head) {
  row = (int)(__umulhi(4u * (unsigned)s, a.share_mul) >> a.share_log);
  head = s - row * a.share;
}

__device__ __attribute__((aligned(64))) const unsigned int bd_da_zero[16] = {};

typedef __attribute__((address_space(3))) void da_lds;

// A staged tile has rows of R bytes; 16-byte chunk ch of row `row` sits at chunk ch ^ f(row). The XOR spreads what is read
// at a time over the banks: by ds_read_b128 four times four neighbouring rows, two groups at one chunk and two at its
// neighbour; by the transposing read two groups of four neighbouring rows, 32 bytes each.
template <int R>
__device__ __forceinline__ int da_off(int row, int ch) {
  const int f = R >= 256 ? (((row & 3) << 2) | ((row >> 2) & 3))
              : R == 128 ? ((((row >> 1) & 1) << 2) | (((row >> 3) & 1) << 1) | ((row >> 2) & 1))
                         : ((row >> 3) & 1) << 1;
  return R * row + 16 * (ch ^ f);
}

typedef __attribute__((address_space(3))) const bf16x8 da_lds_b128;
typedef __attribute__((address_space(3))) s16x4 da_lds_b64;

// Operand reads. Both take one per-lane base (with the tile's address added) and reach every fragment of the tile by an
// XOR and a constant offset: row bits that enter f beside the lane's own (the 4 that tells the halves of 8 rows apart)
// flip one bit, chunk bits above the lane's own flip theirs. One register instead of one per fragment.
// natural rows: lane (g, c) reads row 32 h2 + 8 (c >> 2) + 4 half + (c & 3), chunk 4 ks + g
template <int R>
__device__ __forceinline__ unsigned da_nat_base(int g, int c) { return (unsigned)da_off<R>(8 * (c >> 2) + (c & 3), g); }
template <int R>
__device__ __forceinline__ bf16x8 da_nat(unsigned base, int h2, int half, int ks, int region = 0) {
  const unsigned flip = (R >= 128 && half ? 16u : 0u) | (64u * (unsigned)(ks & (R >= 256 ? 3 : 1)));
  const unsigned add = region + (32 * h2 + 4 * half) * R + (R == 512 ? 256 * (ks >> 2) : 0);
  return *(da_lds_b128*)(size_t)((base ^ flip) + add);
}
// transposed: 8 rows (32 h2 + 8 g ..) x 16 columns (16 dt ..) as an operand whose summed axis runs along the rows
template <int R>
__device__ __forceinline__ unsigned da_tr_base(int g, int c) {
  return (unsigned)(da_off<R>(8 * g + (c >> 2), (c & 3) >> 1) + 8 * (c & 1));
}
template <int R>
__device__ __forceinline__ bf16x8 da_tr(unsigned base, int h2, int dt, int region = 0) {
  const unsigned flip = 32u * (unsigned)(dt & (R >= 256 ? 7 : R == 128 ? 3 : 1));
  const unsigned add = region + 32 * h2 * R + (R == 512 ? 256 * (dt >> 3) : 0);
  union { struct { s16x4 a, b; } s; bf16x8 v; } u;
  u.s.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((da_lds_b64*)(size_t)((base ^ flip) + add));
  u.s.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((da_lds_b64*)(size_t)((base ^ (flip | (R >= 128 ? 16u : 0u))) + add + 4 * R));
  return u.v;
}

// N operand fragments and the products each feeds, with AHEAD fragments read in advance: reads and products keep this order
// (arithmetic may move between them). Left to itself the compiler reads a fragment, waits out the LDS latency and
// multiplies, fragment by fragment, where registers are short (head size 128, 2 x 4096 x 8 heads: forward 432 -> 385 us,
// dkv 819 -> 715; four deep for dkv, 2 and 3 gave 774 and 719).
template <int AHEAD, int N, typename Load, typename Mul>
__device__ __forceinline__ void da_pipe(Load load, Mul mul) {
  constexpr int A = AHEAD < N ? AHEAD : N;
  bf16x8 f[A];
#pragma unroll
  for (int i = 0; i < A; ++i) f[i] = load(i);
  __builtin_amdgcn_sched_barrier(0x6);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    mul(i, f[i % A]);
    if (i + A < N) f[i % A] = load(i + A);
    __builtin_amdgcn_sched_barrier(0x6);
  }
}

// Operands loaded into registers ahead of the staging loop pass through here: the compiler then waits for them once, now.
// Left to itself it puts the wait in front of their first use inside the loop, where every turn would wait for the tile
// just asked for as well (the loads' counter is one, and the compiler does not see the staging).
template <typename V>
__device__ __forceinline__ void da_landed(V& v) { asm volatile("" : "+v"(v)); }

__device__ __forceinline__ void da_dma16(const void* src, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}
// (every lane holds the same pointer; the compiler does not always see that)
__device__ __forceinline__ const unsigned char* da_uniform(const unsigned char* p) {
  const unsigned long long x = (unsigned long long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)x), hi = __builtin_amdgcn_readfirstlane((unsigned)(x >> 32));
  return (const unsigned char*)(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ void da_dma16s(const void* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}

// A value the compiler cannot connect with earlier ones: what is derived from it behind a loop is computed there instead of
// being held in registers through it.
__device__ __forceinline__ int da_again(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Staging of KT rows of R bytes in 1-KiB pieces dealt to NW waves: where in the tile a lane's 16 bytes of piece j land
template <int R, int NW>
struct DaPieces {
  static constexpr int ALL = KT * R / 1024, N = (ALL + NW - 1) / NW;
  static __device__ __forceinline__ int row(int wave, int lane, int j) { return ((wave + NW * j) * 1024 + lane * 16) / R; }
  static __device__ __forceinline__ int chunk(int wave, int lane, int j) {
    const int r = row(wave, lane, j), slot = ((wave + NW * j) * 64 + lane) % (R / 16);
    return (da_off<R>(r, slot) - R * r) >> 4;              // the XOR is its own inverse
  }
  static __device__ __forceinline__ bool any(int wave, int j) { return ALL % NW == 0 || wave + NW * j < ALL; }
};

// rows at base + off[j] (a whole tile inside the tensor, the same offsets tile after tile)
template <int R, int NW>
__device__ __forceinline__ void da_stage_fast(unsigned lds, int wave, const unsigned char* base, const unsigned (&off)[DaPieces<R, NW>::N]) {
  const unsigned char* const from = da_uniform(base);
#pragma unroll
  for (int j = 0; j < DaPieces<R, NW>::N; ++j)
    if (DaPieces<R, NW>::any(wave, j)) da_dma16s(from, off[j], lds + (wave + NW * j) * 1024);
}
// The same for a tile of which some rows are to be zeros: there(row) tells which are fetched. The zeros are written by the
// lanes whose rows are not (the buffer is nobody's until the next barrier, which waits for both).
template <int R, int NW, typename There>
__device__ __forceinline__ void da_stage_some(unsigned lds, int wave, int lane, const unsigned char* base, const unsigned (&off)[DaPieces<R, NW>::N],
                                              There there) {
  const unsigned char* const from = da_uniform(base);
  lane = da_again(lane);                                   // (few tiles come here: nothing of it is held through the loop)
#pragma unroll
  for (int j = 0; j < DaPieces<R, NW>::N; ++j) {
    if (!DaPieces<R, NW>::any(wave, j)) break;
    if (there(DaPieces<R, NW>::row(wave, lane, j))) da_dma16s(from, off[j], lds + (wave + NW * j) * 1024);
    else *(__attribute__((address_space(3))) u32x4*)(size_t)(lds + (wave + NW * j) * 1024 + 16 * lane) = (u32x4){0u, 0u, 0u, 0u};
  }
}
// Strides too far apart for 32-bit offsets: row_ptr(row) = the row's first byte, or null for a row that is to be zeros
template <int R, int NW, typename F>
__device__ __forceinline__ void da_stage(unsigned lds, int wave, int lane, F row_ptr) {
#pragma unroll
  for (int j = 0; j < DaPieces<R, NW>::N; ++j) {
    if (!DaPieces<R, NW>::any(wave, j)) break;
    const unsigned char* p = row_ptr(DaPieces<R, NW>::row(wave, lane, j));
    da_dma16(p ? p + 16 * DaPieces<R, NW>::chunk(wave, lane, j) : (const unsigned char*)bd_da_zero, lds + (wave + NW * j) * 1024);
  }
}

// Key tiles of one key head: both maps' keys and the values
template <int D, int NW>
struct DaKeyStage {
  static constexpr int RK = 2 * D, RV = 4 * D;
  const unsigned char *k0, *k1, *v;
  long long ks, vs;                                        // row strides in bytes
  unsigned ko[DaPieces<RK, NW>::N], vo[DaPieces<RV, NW>::N];
  __device__ __forceinline__ void init(const DaArgs& a, long long bq, long long first, int hk, int wave, int lane) {
    k0 = (const unsigned char*)(a.k + bq * a.ks[0] + first * a.ks[1] + (long long)(2 * hk) * a.ks[2]);
    k1 = k0 + 2 * a.ks[2];
    v = (const unsigned char*)(a.v + bq * a.vs[0] + first * a.vs[1] + (long long)hk * a.vs[2]);
    ks = 2 * a.ks[1]; vs = 2 * a.vs[1];
#pragma unroll
    for (int j = 0; j < DaPieces<RK, NW>::N; ++j)
      ko[j] = (unsigned)ks * DaPieces<RK, NW>::row(wave, lane, j) + 16 * DaPieces<RK, NW>::chunk(wave, lane, j);
#pragma unroll
    for (int j = 0; j < DaPieces<RV, NW>::N; ++j)
      vo[j] = (unsigned)vs * DaPieces<RV, NW>::row(wave, lane, j) + 16 * DaPieces<RV, NW>::chunk(wave, lane, j);
  }
  __device__ __forceinline__ void run(const DaArgs& a, unsigned base, int kt0, unsigned long long vis, int wave, int lane) const {
    if (vis == ~0ull && a.small_strides) {
      da_stage_fast<RK, NW>(base, wave, k0 + ks * kt0, ko);
      da_stage_fast<RK, NW>(base + KT * RK, wave, k1 + ks * kt0, ko);
      da_stage_fast<RV, NW>(base + 2 * KT * RK, wave, v + vs * kt0, vo);
      return;
    }
    if (a.small_strides) {
      auto there = [&](int r) { return ((vis >> r) & 1ull) != 0ull; };
      da_stage_some<RK, NW>(base, wave, lane, k0 + ks * kt0, ko, there);
      da_stage_some<RK, NW>(base + KT * RK, wave, lane, k1 + ks * kt0, ko, there);
      da_stage_some<RV, NW>(base + 2 * KT * RK, wave, lane, v + vs * kt0, vo, there);
      return;
    }
    auto at = [&](const unsigned char* p, long long st) {
      return [=](int r) { return ((vis >> r) & 1ull) ? p + st * (kt0 + r) : (const unsigned char*)nullptr; };
    };
    da_stage<RK, NW>(base, wave, lane, at(k0, ks));
    da_stage<RK, NW>(base + KT * RK, wave, lane, at(k1, ks));
    da_stage<RV, NW>(base + 2 * KT * RK, wave, lane, at(v, vs));
  }
};

__device__ __forceinline__ float da_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

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

struct DaSlot { int row, head; bool ok; };     // (slots behind the last: the last one, ok = false)

__device__ __forceinline__ DaSlot da_slot(const DaArgs& a, int s, int n_slots, int hk) {
  DaSlot r;
  r.ok = s < n_slots;
  s = r.ok ? s : n_slots - 1;
  da_split(a, s, r.row, r.head);
  r.head += hk * a.share;
  return r;
}
__device__ __forceinline__ float da_lam(const DaArgs& a, long long off) {
  return a.lam_f32 ? ((const float*)a.lam)[off] : bd_bf16_to_f32(((const unsigned short*)a.lam)[off]);
}

__device__ __forceinline__ void da_put_dlam(const DaArgs& a, long long at, float v) {
  if (a.dlam_bf16) ((unsigned short*)a.dlam)[at] = bd_f32_to_bf16(v);
  else ((float*)a.dlam)[at] = v;
}

typedef __attribute__((address_space(1))) const unsigned char da_global_byte;      // (a generic load would count as an LDS read)

// one past the last visible key of the sequence (the tiles behind it are not visited); all threads return it
template <int NT>
__device__ __forceinline__ int da_visible_end(const DaArgs& a, int b, int Lk, int tid, int* red) {
  if (!a.mask) return Lk;
  const unsigned char* m = a.mask + b * a.mask_stride;
  int last = 0;
  if (Lk <= 512) {                                         // every wave by itself: all loads in flight, no barrier
    auto scan = [&](auto loads) {
      constexpr int N = decltype(loads)::value;
      unsigned x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = *(da_global_byte*)(m + min(64 * i + (tid & 63), Lk - 1));
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const unsigned long long v = __ballot(x[i] != 0u && 64 * i + (tid & 63) < Lk);
        last = v ? 64 * i + 64 - __builtin_clzll(v) : last;
      }
    };
    if (Lk <= 128) scan(std::integral_constant<int, 2>());
    else scan(std::integral_constant<int, 8>());
    return __builtin_amdgcn_readfirstlane(last);
  }
  for (int j = tid; j < Lk; j += NT) last = m[j] ? j + 1 : last;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o, 64));
  if ((tid & 63) == 0) red[tid >> 6] = last;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) last = max(last, red[w]);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(last);      // (one value: the loops over key tiles count on the scalar unit)
}

// mask byte of the lane's key of a tile (0 past the end)
__device__ __forceinline__ unsigned da_mask_byte(const DaArgs& a, int b, int key, int end) {
  if (key >= end) return 0u;
  if (!a.mask) return 1u;
  return *(da_global_byte*)(a.mask + b * a.mask_stride + key);
}

// Workgroups are handed to the 8 XCDs in turn (blockIdx & 7). The blocks of one (sequence, key head) group share an XCD, so
// that they find the group's rows in its L2. Many groups: dealt to the XCDs one by one (ragged sequences then load all XCDs
// alike); few: the list of all blocks is cut into eight contiguous parts. False: no work for this workgroup.
__device__ __forceinline__ bool da_block(int n_blk, int n_heads, int seqs, int& blk, int& hk, int& b) {
  const int groups = n_heads * seqs, xcd = blockIdx.x & 7, j = blockIdx.x >> 3;
  int grp;
  if (groups % 8 == 0 || groups >= 64) {
    grp = (j / n_blk) * 8 + xcd;
    blk = j % n_blk;
    if (grp >= groups) return false;
  } else {
    const int n_all = groups * n_blk, q = n_all >> 3, rr = n_all & 7;
    if (j >= q + (xcd < rr ? 1 : 0)) return false;
    const int lin = (xcd < rr ? xcd * (q + 1) : rr * (q + 1) + (xcd - rr) * q) + j;
    blk = lin % n_blk;
    grp = lin / n_blk;
  }
  // (the divisions ran on the vector unit: tell the compiler that every lane holds the same)
  blk = __builtin_amdgcn_readfirstlane(blk);
  hk = __builtin_amdgcn_readfirstlane(grp % n_heads);
  b = __builtin_amdgcn_readfirstlane(grp / n_heads);
  return true;
}
inline long long da_grid(long long n_blk, long long groups) { return n_blk * ((groups + 7) / 8) * 8; }

// rows first .. end - 1 of heads head0 .. of width W, every 32 bits of them set to `word`
__device__ __forceinline__ void da_fill(unsigned short* p, const long long* st, int first, int end, unsigned word, int head0, int heads, int W,
                                        int tid, int nt) {
  const int per = heads * (W / 8);
  for (long long i = tid; i < (long long)(end - first) * per; i += nt) {
    const int row = first + (int)(i / per), r = (int)(i % per);
    *(u32x4*)(p + row * st[1] + (long long)(head0 + r / (W / 8)) * st[2] + 8 * (r % (W / 8))) = (u32x4){word, word, word, word};
  }
}
// Packed rows that no sequence's workgroups write (one workgroup a head, all NT threads): zeros before the first and behind
// the last sequence, NaN (no silence) in a sequence longer than announced, from its row Lq on.
template <int NT, typename Fill>
__device__ __forceinline__ void da_unclaimed(const DaArgs& a, int tid, Fill fill) {
  fill(0, min(max(a.cu[0], 0), a.total), 0u);
  fill(min(max(a.cu[a.B], 0), a.total), a.total, 0u);
  int longer = 0;
  for (int i = tid; i < a.B; i += NT) longer |= min(a.cu[i + 1], a.total) - max(a.cu[i], 0) > a.Lq;
  const int n = __syncthreads_or(longer) ? a.B : 0;
  for (int i = 0; i < n; ++i) {
    const int lo = min(max(a.cu[i], 0), a.total), hi = min(max(a.cu[i + 1], lo), a.total);
    if (hi - lo > a.Lq) fill(lo + a.Lq, hi, 0x7fc07fc0u);
  }
}

// =====================================================================================
// Forward. Waves work in pairs: wave 2 w + m holds map m of the 16 QB slots of query group w (NQG groups in a
// workgroup). Split over keys (n_split > 1): each split leaves its unnormalised sums, maximum and normaliser.
// Head size 128 (2 x 4096 tokens, 8 heads over 4: 391 us, 1.05 PFLOP/s): matrix cores busy 52 % of the cycles, vector units
// 44 %: the exponentials of one wave of a SIMD run under the products of the other. Head sizes 32 and 64: vector units 66 %
// and 56 % busy, matrix cores 19 % and 11 %, so neither is full: about 4 vector instructions a score in the loop and those
// around it (many short sequences), each waiting for the one before with four waves a SIMD to hide it.
// =====================================================================================
template <int D, int QB, int NQG, int OCC, bool TWO>
__global__ __launch_bounds__(128 * NQG, OCC) void da_fwd_kernel(DaArgs a) {
  constexpr int E = 2 * D, AF = D == 128 ? 3 : 6, KS = D / 32, DT = E / 16, NW = 2 * NQG, RK = 2 * D, RV = 2 * E;
  constexpr int TILE = KT * (2 * RK + RV), SLOTS = 16 * QB * NQG;
  extern __shared__ __attribute__((aligned(1024))) unsigned char da_smem[];
  __shared__ int red[NW];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int map = wave & 1, grp = wave >> 1;
  const int g = lane >> 4, c = lane & 15;
  int blk, hk, b;
  if (!da_block(a.n_blk * a.n_split, a.Hkv, a.B + (a.cu ? 1 : 0), blk, hk, b)) return;
  const int split = blk % a.n_split;
  blk /= a.n_split;
  if (a.cu && b == a.B) {                                  // (packed: one more sequence, the rows of none)
    if (blk == 0)
      da_unclaimed<64 * NW>(a, tid, [&](int first, int end, unsigned word) {
        da_fill(a.out, a.os, first, end, word, hk * a.share, a.share, E, tid, 64 * NW);
      });
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
  const int s0 = blk * SLOTS + grp * 16 * QB + c;
  bf16x8 qf[QB][KS];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const DaSlot sl = da_slot(a, s0 + 16 * qb, n_slots, hk);
    const unsigned short* qp = a.q + bq * a.qs[0] + (sp.q0 + sl.row) * a.qs[1] + (2 * sl.head + map) * a.qs[2] + 8 * g;
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
  const float scale2 = a.scale * LOG2E, slack = 8.f / scale2;

  DaKeyStage<D, NW> keys;
  keys.init(a, bq, sp.k0, hk, wave, lane);
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) da_landed(qf[qb][ks]);
  const unsigned lds0 = (unsigned)(size_t)(da_lds*)da_smem;
  const unsigned kbase = da_nat_base<RK>(g, c) + map * KT * RK, vbase = da_tr_base<RV>(g, c) + 2 * KT * RK;
  unsigned mb = da_mask_byte(a, b, kbeg + lane, kend);
  unsigned long long vis = __ballot(mb != 0u);
  if (kbeg < kend) keys.run(a, lds0, kbeg, vis, wave, lane);
  mb = da_mask_byte(a, b, kbeg + KT + lane, kend);
  unsigned cur = lds0, other = lds0 + TILE;
  for (int kt0 = kbeg; kt0 < kend; kt0 += KT) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // this tile is there, nobody reads the other buffer
    const unsigned long long vis_next = __ballot(mb != 0u);
    mb = da_mask_byte(a, b, kt0 + 2 * KT + lane, kend);
    if (kt0 + KT < kend) keys.run(a, other, kt0 + KT, vis_next, wave, lane);
    const unsigned kb = cur + kbase, vb = cur + vbase;

    // S^T: s[qb][t][r] <-> key 32 (t >> 1) + 8 g + 4 (t & 1) + r of the tile, slot c of block qb
    f32x4 s[QB][4];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int t = 0; t < 4; ++t) s[qb][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    da_pipe<AF, 4 * KS>([&](int i) { return da_nat<RK>(kb, i / KS >> 1, i / KS & 1, i % KS); },
                    [&](int i, bf16x8 kf) {
#pragma unroll
                      for (int qb = 0; qb < QB; ++qb)
                        s[qb][i / KS] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[qb][i % KS], s[qb][i / KS], 0, 0, 0);
                    });
    bf16x8 pf[QB][2], pl[QB][2];
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
      // (the IEEE maximum of three values is one instruction here; fmaxf would first quiet each product's result)
      float mloc = da_max(s[qb][0][0], s[qb][0][1]);
#pragma unroll
      for (int i = 2; i < 16; i += 2) mloc = da_max(mloc, da_max(s[qb][i >> 2][i & 3], s[qb][i >> 2][(i & 3) + 1]));
      // The reference of the exponentials follows the maximum only when a score passes it by 2^8: weights then reach 2^8 at
      // most (no less exact in bf16 and fp32), and almost every tile goes without the exchange between a slot's four lanes
      // and without rescaling.
      if (__any(mloc > m_run[qb] + slack)) {
        mloc = fmaxf(mloc, __shfl_xor(mloc, 16, 64));
        mloc = fmaxf(mloc, __shfl_xor(mloc, 32, 64));
        const float m_new = fmaxf(m_run[qb], mloc);
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_run[qb] - m_new) * scale2);
        m_run[qb] = m_new;
        l_run[qb] *= alpha;
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
          // Weights to bf16 for the second product (half a step: 2^-8 of each weight; the normaliser keeps them in fp32). A few
          // rows split over the keys wait for memory, not for products: there a second bf16 holds what the first left out
          // (2^-16), for 23.2 -> 23.8 us at one row against 65 521 keys; with all keys in one workgroup it would be 16.9 ->
          // 18.8 us (2 rows against 512 keys), and the large products would grow by half.
          const __bf16 hi = (__bf16)p;
          pf[qb][t >> 1][4 * (t & 1) + r] = hi;
          if (TWO) pl[qb][t >> 1][4 * (t & 1) + r] = (__bf16)(p - (float)hi);
        }
    }
    // O^T += V^T P^T
    da_pipe<AF, 2 * DT>([&](int i) { return da_tr<RV>(vb, i & 1, i >> 1); },
                    [&](int i, bf16x8 vf) {
#pragma unroll
                      for (int qb = 0; qb < QB; ++qb) {
                        o[qb][i >> 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[qb][i & 1], o[qb][i >> 1], 0, 0, 0);
                        if (TWO) o[qb][i >> 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl[qb][i & 1], o[qb][i >> 1], 0, 0, 0);
                      }
                    });
    vis = vis_next;
    const unsigned sw = cur; cur = other; other = sw;
  }
  // lane holds O[slot c of block qb][16 dt + 4 g + r] of its map
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    l_run[qb] += __shfl_xor(l_run[qb], 16, 64);
    l_run[qb] += __shfl_xor(l_run[qb], 32, 64);
  }
  const int s1 = da_again(s0), g1 = (da_again(lane) >> 4);
  if (a.n_split > 1) {
    const long long pb = ((long long)(b * a.Hkv + hk) * a.n_blk + blk) * a.n_split + split;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      if (s1 + 16 * qb >= n_slots) continue;
      const long long at = (pb * 2 + map) * SLOTS + (s1 + 16 * qb - blk * SLOTS);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *(f32x4*)(a.part + at * E + 16 * dt + 4 * g1) = o[qb][dt];
      if (g1 == 0) *(f32x2*)(a.part_ml + 2 * at) = (f32x2){m_run[qb] * scale2, l_run[qb]};
    }
    return;
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float l = l_run[qb];
    const bool any = l > 0.f || l != l;
    const float inv = any ? 1.0f / l : 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[qb][dt][r] *= inv;
    if (a.lse) {
      const DaSlot sl = da_slot(a, s1 + 16 * qb, n_slots, hk);
      const long long rh = (bq * a.Lq + sp.q0 + sl.row) * a.H + sl.head;       // row and head, counted through the batch
      if (sl.ok && g1 == 0)                // base 2, for the scaled scores; +inf: no visible key, every weight 2^-inf = 0
        a.lse[2 * rh + map] = any ? m_run[qb] * scale2 + __log2f(l) : INFINITY;
      if (sl.ok && a.maps) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *(f32x4*)(a.maps + (2 * rh + map) * E + 16 * dt + 4 * g1) = o[qb][dt];
      }
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
      const DaSlot sl = da_slot(a, s1 + 16 * qb, n_slots, hk);
      if (!sl.ok) continue;
      const float lam = da_lam(a, bq * a.ls[0] + (sp.q0 + sl.row) * a.ls[1] + sl.head * a.ls[2]);
      unsigned short* op = a.out + bq * a.os[0] + (sp.q0 + sl.row) * a.os[1] + sl.head * a.os[2] + 4 * g1;
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

// first of a slot's partial sums: [sequence and key head][block of slots][split][map][slot of the block]
__device__ __forceinline__ long long da_part(const DaArgs& a, int b, int hk, int slot) {
  const int blk = slot / a.per;
  return ((long long)(b * a.Hkv + hk) * a.n_blk + blk) * a.n_split * 2 * a.per + (slot - blk * a.per);
}

// four columns of a slot whose maps' sums, maxima and normalisers are joined
template <int D>
__device__ __forceinline__ void da_joined(const DaArgs& a, int b, const DaSlot& sl, long long rh, int col, f32x4 (&r)[2], const float (&top)[2],
                                          const float (&l)[2]) {
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const bool any = l[m] > 0.f || l[m] != l[m];
    const float inv = any ? 1.0f / l[m] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[m][e] *= inv;
    if (a.maps) *(f32x4*)(a.maps + (2 * rh + m) * 2 * D + col) = r[m];
    if (a.lse && col == 0) a.lse[2 * rh + m] = any ? top[m] + __log2f(l[m]) : INFINITY;
  }
  const float lam = da_lam(a, b * a.ls[0] + sl.row * a.ls[1] + sl.head * a.ls[2]);
  u32x2 w;
  w[0] = bd_pack_bf16x2(r[0][0] - lam * r[1][0], r[0][1] - lam * r[1][1]);
  w[1] = bd_pack_bf16x2(r[0][2] - lam * r[1][2], r[0][3] - lam * r[1][3]);
  *(u32x2*)(a.out + b * a.os[0] + sl.row * a.os[1] + sl.head * a.os[2] + col) = w;
}

// Joins more than 16 key splits of one slot, 16 columns a workgroup: waves 2 m and 2 m + 1 add up map m, 16 splits at a time
// each with 4 lanes across the columns, in a fixed order. Bound by latency (one row, 65 521 keys, 4 x 4 heads of 64, 64
// splits: 1 MB of partial sums, 4.7 us): what a thread adds up is asked for before the splits' maxima and normalisers are
// worked into weights, and many small workgroups wait at once.
constexpr int JOIN_COLS = 16, JOIN_SPLITS = 256, JOIN_LANES = 16;
template <int D>
__global__ __launch_bounds__(256) void da_join_kernel(DaArgs a) {
  constexpr int E = 2 * D, CB = E / JOIN_COLS, N = JOIN_SPLITS / 32;
  __shared__ float wt[2][JOIN_SPLITS], red[2][2][4];
  __shared__ f32x4 sum[4][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slot = blockIdx.x / CB, col = (blockIdx.x % CB) * JOIN_COLS + 4 * (lane & 3), hk = blockIdx.y, b = blockIdx.z;
  const DaSlot sl = da_slot(a, slot, a.Lq * a.share, hk);
  const long long rh = ((long long)b * a.Lq + sl.row) * a.H + sl.head;
  const long long at0 = da_part(a, b, hk, slot);
  const int map = wave >> 1, s0 = (wave & 1) * 16 + (lane >> 2);
  f32x4 x[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (s0 + 32 * i < a.n_split) x[i] = *(const f32x4*)(a.part + (at0 + (long long)(2 * (s0 + 32 * i) + map) * a.per) * E + col);
  f32x2 ml[2] = {{-INFINITY, 0.f}, {-INFINITY, 0.f}};
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (tid < a.n_split) ml[m] = *(const f32x2*)(a.part_ml + 2 * (at0 + (long long)(2 * tid + m) * a.per));
    const float mx = bd_wave_max(ml[m][0]);
    if (lane == 0) red[0][m][wave] = mx;
  }
  __syncthreads();
  float top[2], l[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    top[m] = fmaxf(fmaxf(red[0][m][0], red[0][m][1]), fmaxf(red[0][m][2], red[0][m][3]));
    // a split without a visible key weighs nothing
    const float w = ml[m][1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[m][0] - top[m]);
    wt[m][tid] = w;
    const float ls = bd_wave_sum(w * ml[m][1]);
    if (lane == 0) red[1][m][wave] = ls;
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < 2; ++m) l[m] = (red[1][m][0] + red[1][m][1]) + (red[1][m][2] + red[1][m][3]);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (s0 + 32 * i < a.n_split) {
      const float w = wt[map][s0 + 32 * i];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += w == 0.f ? 0.f : w * x[i][e];
    }
#pragma unroll
  for (int s = 4; s < 64; s *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], s, 64);
  if (lane < 4) sum[wave][lane] = o;
  __syncthreads();
  if (tid >= 4) return;
  f32x4 r[2];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) r[m][e] = sum[2 * m][tid][e] + sum[2 * m + 1][tid][e];
  da_joined<D>(a, b, sl, rh, col, r, top, l);
}

// The same for at most 16 splits (many slots: the launch is bound by the partial sums' way through memory): a wave takes 16
// (slot, split) pairs, four lanes across 16 columns each, and adds up by exchanges alone (2048 slots, 2 splits of 64-wide
// heads: 8.3 us).
template <int D>
__global__ __launch_bounds__(256) void da_join_few_kernel(DaArgs a) {
  constexpr int E = 2 * D, CB = E / JOIN_COLS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hk = blockIdx.y, b = blockIdx.z;
  int lanes = 2;                                           // lanes (of four) that share a slot
  while (lanes < a.n_split) lanes *= 2;
  const int n_slots = a.Lq * a.share, pair = lane >> 2, split = pair & (lanes - 1), here = JOIN_LANES / lanes;
  const int slot = ((int)(blockIdx.x / CB) * 4 + wave) * here + pair / lanes, col = (int)(blockIdx.x % CB) * JOIN_COLS + 4 * (lane & 3);
  const DaSlot sl = da_slot(a, slot, n_slots, hk);
  const long long rh = ((long long)b * a.Lq + sl.row) * a.H + sl.head;
  const long long at0 = da_part(a, b, hk, min(slot, n_slots - 1));
  f32x4 x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  f32x2 ml[2] = {{-INFINITY, 0.f}, {-INFINITY, 0.f}};
#pragma unroll
  for (int m = 0; m < 2; ++m)
    if (split < a.n_split) {
      const long long at = at0 + (long long)(2 * split + m) * a.per;
      ml[m] = *(const f32x2*)(a.part_ml + 2 * at);
      x[m] = *(const f32x4*)(a.part + at * E + col);
    }
  float top[2], l[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    top[m] = ml[m][0];
    for (int s = 4; s < 4 * lanes; s *= 2) top[m] = fmaxf(top[m], __shfl_xor(top[m], s, 64));
    const float w = ml[m][1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[m][0] - top[m]);
    l[m] = w * ml[m][1];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[m][e] = w == 0.f ? 0.f : w * x[m][e];
    for (int s = 4; s < 4 * lanes; s *= 2) {
      l[m] += __shfl_xor(l[m], s, 64);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[m][e] += __shfl_xor(x[m][e], s, 64);
    }
  }
  if (split == 0 && sl.ok) da_joined<D>(a, b, sl, rh, col, x, top, l);
}

// =====================================================================================
// Backward, query side: dQ and what the key side needs of each slot (stats: lse1, lse2, delta1, delta2, lam, scale of
// dK), dlam. A wave owns 16 QB slots and both of their maps (dP = dO V^T is shared). delta_m comes from the forward's
// fp32 maps (dO . O_m) or, where none were kept, from a first walk over the keys (SHORT: from what the only walk leaves
// in registers): sums of the very P and dP that form dS. From a bf16-rounded O it would miss sum_j dS_ij = 0 by 2^-9 of
// |dO||O| for all keys alike, as large as dS itself where attention is nearly uniform. dlam is always -sum_j P2 dP of the
// walk: the fp32 maps hold the forward's bf16 weights (1.7e-3 of a row), which a weight per head, summed over rows that
// cancel, does not bear (5.9e-3 of 36 x 739 rows' sum, now the 2^-8 of its own rounding; one fma a pair, 1 % of dq at
// head size 32, 3 % at 128). Head size 128 as above: 440 us, 0.94 PFLOP/s, matrix cores busy 45 %, vector units 42 %. At 128
// keys of 64-wide heads the matrix cores are busy 10 % of the cycles and the vector units 36 %: it waits for its operands and
// for dependent instructions (few tiles a workgroup).
// =====================================================================================
template <int D, int QB, int NW, int OCC, bool SHORT>
__global__ __launch_bounds__(64 * NW, OCC) void da_bwd_dq_kernel(DaArgs a) {
  constexpr int E = 2 * D, AQ = D == 32 ? 6 : 4, KS = D / 32, ES = E / 32, DT = D / 16, RK = 2 * D, RV = 2 * E;
  constexpr int TILE = KT * (2 * RK + RV), SLOTS = 16 * QB * NW;
  extern __shared__ __attribute__((aligned(1024))) unsigned char da_smem[];
  __shared__ int red[NW];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  int blk, hk, b;
  if (!da_block(a.n_blk, a.Hkv, a.B + (a.cu ? 1 : 0), blk, hk, b)) return;
  if (a.cu && b == a.B) {
    if (blk == 0)
      da_unclaimed<64 * NW>(a, tid, [&](int first, int end, unsigned word) {
        if (a.dq) da_fill(a.dq, a.dqs, first, end, word, 2 * hk * a.share, 2 * a.share, D, tid, 64 * NW);
        for (long long i = tid; i < (long long)(end - first) * a.share; i += 64 * NW)
          da_put_dlam(a, (first + i / a.share) * a.H + hk * a.share + i % a.share, word ? __uint_as_float(0x7fc00000u) : 0.f);
      });
    return;
  }
  const DaSpan sp = da_span(a, b);
  const int n_slots = sp.Lq * a.share;
  if (blk * SLOTS >= n_slots) return;
  const long long bq = a.cu ? 0 : b;
  const int kend = da_visible_end<64 * NW>(a, b, sp.Lk, tid, red);

  const int s0 = blk * SLOTS + wave * 16 * QB + c;
  bf16x8 qf[QB][2][KS], dof[QB][ES];
  float lse[QB][2], dl[QB][2];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const DaSlot sl = da_slot(a, s0 + 16 * qb, n_slots, hk);
    const long long rh = (bq * a.Lq + sp.q0 + sl.row) * a.H + sl.head;
    const unsigned short* dp = a.dout + bq * a.dos[0] + (sp.q0 + sl.row) * a.dos[1] + sl.head * a.dos[2] + 8 * g;
#pragma unroll
    for (int ks = 0; ks < ES; ++ks) dof[qb][ks] = *(const bf16x8*)(dp + 32 * ks);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const unsigned short* qp = a.q + bq * a.qs[0] + (sp.q0 + sl.row) * a.qs[1] + (2 * sl.head + m) * a.qs[2] + 8 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[qb][m][ks] = *(const bf16x8*)(qp + 32 * ks);
      lse[qb][m] = a.lse[2 * rh + m];
      dl[qb][m] = 0.f;
      if (a.maps) {
        const float* op = a.maps + (2 * rh + m) * E + 8 * g;
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

  DaKeyStage<D, NW> keys;
  keys.init(a, bq, sp.k0, hk, wave, lane);
  const unsigned lds0 = (unsigned)(size_t)(da_lds*)da_smem;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
#pragma unroll
    for (int ks = 0; ks < ES; ++ks) da_landed(dof[qb][ks]);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      da_landed(lse[qb][m]);
      da_landed(dl[qb][m]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) da_landed(qf[qb][m][ks]);
    }
  }
  const unsigned knat = da_nat_base<RK>(g, c), ktr = da_tr_base<RK>(g, c), vnat = da_nat_base<RV>(g, c) + 2 * KT * RK;
  // scores of 16 keys (half a 32-key group) against the wave's slots, and dP; masked keys' scores are -inf
  auto scores = [&](unsigned kn, unsigned vn, int half, unsigned long long vis32, f32x4 (&s)[QB][2], f32x4 (&dp)[QB]) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) s[qb][0] = s[qb][1] = dp[qb] = (f32x4){0.f, 0.f, 0.f, 0.f};
    // fragments: keys of map 0 and 1 in turn, then the values
    da_pipe<AQ, 2 * KS + ES>([&](int i) { return i < 2 * KS ? da_nat<RK>(kn, 0, half, i >> 1, (i & 1) * KT * RK) : da_nat<RV>(vn, 0, half, i - 2 * KS); },
                         [&](int i, bf16x8 x) {
#pragma unroll
                           for (int qb = 0; qb < QB; ++qb) {
                             if (i < 2 * KS) s[qb][i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, qf[qb][i & 1][i >> 1], s[qb][i & 1], 0, 0, 0);
                             else dp[qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, dof[qb][i - 2 * KS], dp[qb], 0, 0, 0);
                           }
                         });
    if ((unsigned)vis32 != ~0u) {
      const unsigned m4 = (unsigned)(vis32 >> (8 * g + 4 * half)) & 0xfu;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!((m4 >> r) & 1u)) s[qb][0][r] = s[qb][1][r] = -INFINITY;        // weight 2^-inf = 0 (dP of a zero row is 0)
    }
  };
  // (dS goes to bf16 as the product's operand: half a step is 2^-8 of each, and its sum over the keys misses zero by no more)
  auto add_dq = [&](unsigned kt, const bf16x8 (&dsf)[QB][2]) {                 // dQ^T += K^T dS^T
    da_pipe<AQ, 2 * DT>([&](int i) { return da_tr<RK>(kt, 0, i >> 1, (i & 1) * KT * RK); },
                    [&](int i, bf16x8 x) {
#pragma unroll
                      for (int qb = 0; qb < QB; ++qb)
                        acc[qb][i & 1][i >> 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, dsf[qb][i & 1], acc[qb][i & 1][i >> 1], 0, 0, 0);
                    });
  };
  int seen = 0;                                            // keys that the mask leaves
  float dm[QB];                                            // dP . P2 of the rows, for dlam
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) dm[qb] = 0.f;
  // last: dQ is summed; only: dlam's sums, delta is there from the maps; neither: delta (and dlam with it)
  auto walk_keys = [&](auto last, auto only) {
    constexpr bool LAST = decltype(last)::value, ONLY = decltype(only)::value;
    unsigned mb = da_mask_byte(a, b, lane, kend);
    unsigned long long vis = __ballot(mb != 0u);
    __syncthreads();                                       // (second walk: nobody reads the first one's last tile)
    unsigned cur = lds0, other = lds0 + TILE;
    if (kend > 0) keys.run(a, cur, 0, vis, wave, lane);
    mb = da_mask_byte(a, b, KT + lane, kend);
    for (int kt0 = 0; kt0 < kend; kt0 += KT) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const unsigned long long vis_next = __ballot(mb != 0u);
      mb = da_mask_byte(a, b, kt0 + 2 * KT + lane, kend);
      if (kt0 + KT < kend) keys.run(a, other, kt0 + KT, vis_next, wave, lane);
      if (!LAST || ONLY) seen += __popcll(vis);            // (in the first walk)
#pragma unroll 1                                           // (unrolled, the scheduler reads ahead more than the registers hold)
      for (int h2 = 0; h2 < 2; ++h2) {                     // 32 keys
        const unsigned kn = cur + knat + 32 * RK * h2, kt = cur + ktr + 32 * RK * h2, vn = cur + vnat + 32 * RV * h2;
        bf16x8 dsf[QB][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          f32x4 s[QB][2], dp[QB];
          scores(kn, vn, half, vis >> (32 * h2), s, dp);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float p = __builtin_amdgcn_exp2f(s[qb][m][r] * scale2 - lse[qb][m]);
                if (ONLY && m == 1) dm[qb] += p * dp[qb][r];
                if (LAST) dsf[qb][m][4 * half + r] = (__bf16)(p * (dp[qb][r] - dl[qb][m]));
                else if (!ONLY) dl[qb][m] += p * dp[qb][r];
              }
        }
        if (LAST) add_dq(kt, dsf);
      }
      vis = vis_next;
      const unsigned sw = cur; cur = other; other = sw;
    }
  };
  auto join = [&](float& x) {                              // the lanes that share a slot
    x += __shfl_xor(x, 16, 64);
    x += __shfl_xor(x, 32, 64);
  };
  auto join_delta = [&] {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      join(dl[qb][0]);
      join(dl[qb][1]);
      dm[qb] = dl[qb][1];
    }
  };
  if constexpr (SHORT) {                                   // both tiles stay in LDS, their weights and dP in registers
    f32x4 p[2][2][2][QB][2], dp[2][2][2][QB];              // [tile][32 keys][16 of them]
    unsigned long long vis[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      vis[t] = __ballot(da_mask_byte(a, b, KT * t + lane, kend) != 0u);
      seen += __popcll(vis[t]);
      if (KT * t < kend) keys.run(a, lds0 + t * TILE, KT * t, vis[t], wave, lane);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (KT * t >= kend) continue;
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          f32x4 (&s)[QB][2] = p[t][h2][half];
          f32x4 (&d)[QB] = dp[t][h2][half];
          scores(lds0 + t * TILE + knat + 32 * RK * h2, lds0 + t * TILE + vnat + 32 * RV * h2, half, vis[t] >> (32 * h2), s, d);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                s[qb][m][r] = __builtin_amdgcn_exp2f(s[qb][m][r] * scale2 - lse[qb][m]);
                dl[qb][m] += s[qb][m][r] * d[qb][r];
              }
        }
    }
    join_delta();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (KT * t >= kend || !a.dq) continue;
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        bf16x8 dsf[QB][2];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 8; ++i) dsf[qb][m][i] = (__bf16)(p[t][h2][i >> 2][qb][m][i & 3] * (dp[t][h2][i >> 2][qb][i & 3] - dl[qb][m]));
        add_dq(lds0 + t * TILE + ktr + 32 * RK * h2, dsf);
      }
    }
  } else {
    if (a.maps) {
      if (a.dq) walk_keys(std::true_type(), std::true_type());
      else walk_keys(std::false_type(), std::true_type());
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) join(dm[qb]);
    } else {
      walk_keys(std::false_type(), std::false_type());
      join_delta();
      if (a.dq) walk_keys(std::true_type(), std::false_type());
    }
  }
  // One key alone has weight 1 whatever its score: dQ and dK are exact zeros, where 2^(s - lse) rounds beside 1
  const float scale = seen == 1 ? 0.f : a.scale;
  const int s1 = da_again(s0), g1 = da_again(lane) >> 4;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const DaSlot sl = da_slot(a, s1 + 16 * qb, n_slots, hk);
    if (!sl.ok) continue;
    const long long rh = (bq * a.Lq + sp.q0 + sl.row) * a.H + sl.head;
    const float lam = da_lam(a, bq * a.ls[0] + (sp.q0 + sl.row) * a.ls[1] + sl.head * a.ls[2]);
    if (g1 == 0) {
      *(f32x4*)(a.stats + 8 * rh) = (f32x4){lse[qb][0], lse[qb][1], dl[qb][0], dl[qb][1]};
      *(f32x2*)(a.stats + 8 * rh + 4) = (f32x2){lam, scale};
      da_put_dlam(a, rh, -dm[qb]);
    }
    if (!a.dq) continue;                                   // q needs no gradient
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const float f = m ? -lam * scale : scale;
      unsigned short* op = a.dq + bq * a.dqs[0] + (sp.q0 + sl.row) * a.dqs[1] + (2 * sl.head + m) * a.dqs[2] + 4 * g1;
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
// Backward, key side: a workgroup owns 16 KB NW keys of one key head and walks the query slots of all heads that share it.
// Head size 128 as above: 713 us, 0.77 PFLOP/s. Every operand fragment read from LDS feeds one product (a wave cannot hold the
// sums, keys and values of 32 keys beside a second wave on its SIMD): 64 KB a wave for 32 slots, at 128 bytes a cycle 4100
// cycles a CU for 2048 of products. Waves of 32 keys alone on their SIMD lose more to what they cannot overlap (above).
// =====================================================================================
template <int D, int KB, int NW, int OCC>
__global__ __launch_bounds__(64 * NW, OCC) void da_bwd_dkv_kernel(DaArgs a) {
  constexpr int E = 2 * D, AK = D == 128 ? 4 : 6, KS = D / 32, ES = E / 32, DT = D / 16, ET = E / 16, RK = 2 * D, RV = 2 * E;
  constexpr int TILE = KT * (2 * RK + RV + 32), KEYS = 16 * KB * NW;
  extern __shared__ __attribute__((aligned(1024))) unsigned char da_smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  int blk, hk, b;
  if (!da_block(a.n_blk, a.Hkv, a.B + (a.cu ? 1 : 0), blk, hk, b)) return;
  if (a.cu && b == a.B) {
    if (blk == 0)
      da_unclaimed<64 * NW>(a, tid, [&](int first, int end, unsigned word) {
        da_fill(a.dk, a.dks, first, end, word, 2 * hk, 2, D, tid, 64 * NW);
        da_fill(a.dv, a.dvs, first, end, word, hk, 1, E, tid, 64 * NW);
      });
    return;
  }
  const DaSpan sp = da_span(a, b);
  if (blk * KEYS >= sp.Lk) return;
  const long long bq = a.cu ? 0 : b;
  const int n_slots = sp.Lq * a.share;
  const int k0 = blk * KEYS + wave * 16 * KB + c;
  bool live = false;
  bf16x8 kf[KB][2][KS], vf[KB][ES];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int key = min(k0 + 16 * kb, sp.Lk - 1);
    live = live || (k0 + 16 * kb < sp.Lk && (!a.mask || a.mask[b * a.mask_stride + key] != 0));
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
  // Slot tiles: row s / share, head hk * share + s % share. Where share divides the tile a lane's offsets are the same for
  // every whole tile and the base moves by KT / share rows.
  typedef DaPieces<RK, NW> PQ;
  typedef DaPieces<RV, NW> PD;
  const unsigned char* const qb0 = (const unsigned char*)(a.q + bq * a.qs[0] + sp.q0 * a.qs[1] + (long long)(2 * hk * a.share) * a.qs[2]);
  const unsigned char* const db0 = (const unsigned char*)(a.dout + bq * a.dos[0] + sp.q0 * a.dos[1] + (long long)(hk * a.share) * a.dos[2]);
  const unsigned char* const sb0 = (const unsigned char*)(a.stats + 8 * ((bq * a.Lq + sp.q0) * a.H + hk * a.share));
  const bool even = a.small_strides && KT % a.share == 0;
  unsigned qo[PQ::N], dob[PD::N], so;
  {
    int row, head;
#pragma unroll
    for (int j = 0; j < PQ::N; ++j) {
      da_split(a, PQ::row(wave, lane, j), row, head);
      qo[j] = (unsigned)(2 * a.qs[1]) * row + (unsigned)(4 * a.qs[2]) * head + 16 * PQ::chunk(wave, lane, j);
    }
#pragma unroll
    for (int j = 0; j < PD::N; ++j) {
      da_split(a, PD::row(wave, lane, j), row, head);
      dob[j] = (unsigned)(2 * a.dos[1]) * row + (unsigned)(2 * a.dos[2]) * head + 16 * PD::chunk(wave, lane, j);
    }
    da_split(a, lane, row, head);
    so = (unsigned)(row * a.H + head) * 32 + 16 * (wave & 1);
  }
  auto stage = [&](int t0, unsigned base) {
    if (even && t0 + KT <= n_slots) {
      const int row0 = t0 / a.share;
      const unsigned char* const q0 = qb0 + 2 * a.qs[1] * row0;
      da_stage_fast<RK, NW>(base, wave, q0, qo);
      da_stage_fast<RK, NW>(base + KT * RK, wave, q0 + 2 * a.qs[2], qo);
      da_stage_fast<RV, NW>(base + 2 * KT * RK, wave, db0 + 2 * a.dos[1] * row0, dob);
      if (wave < 2) da_dma16s(da_uniform(sb0 + 32ll * row0 * a.H), so, base + KT * (2 * RK + RV) + wave * 1024);
      return;
    }
    auto at = [&](const unsigned char* p, long long rs, long long hs) {
      return [=](int r) {
        int row, head;
        const int s = da_again(t0 + r);                    // (a last tile's: nothing of it is held through the loop)
        da_split(a, s, row, head);
        return s < n_slots ? p + row * rs + head * hs : (const unsigned char*)nullptr;
      };
    };
    da_stage<RK, NW>(base, wave, lane, at(qb0, 2 * a.qs[1], 4 * a.qs[2]));
    da_stage<RK, NW>(base + KT * RK, wave, lane, at(qb0 + 2 * a.qs[2], 2 * a.qs[1], 4 * a.qs[2]));
    da_stage<RV, NW>(base + 2 * KT * RK, wave, lane, at(db0, 2 * a.dos[1], 2 * a.dos[2]));
    if (wave < 2) {                                        // the slots' statistics: lane = slot, 16 bytes a wave
      const unsigned char* src = at(sb0, 32ll * a.H, 32)(lane);
      da_dma16(src ? src + 16 * wave : (const unsigned char*)bd_da_zero, base + KT * (2 * RK + RV) + wave * 1024);
    }
  };
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
    for (int ks = 0; ks < ES; ++ks) da_landed(vf[kb][ks]);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) da_landed(kf[kb][m][ks]);
  }
  const unsigned qnat = da_nat_base<RK>(g, c), qtr = da_tr_base<RK>(g, c);
  const unsigned dnat = da_nat_base<RV>(g, c) + 2 * KT * RK, dtr = da_tr_base<RV>(g, c) + 2 * KT * RK;
  if (__syncthreads_or(live)) {                            // no visible key in this workgroup: every gradient is zero
    unsigned cur = lds0, other = lds0 + TILE;
    stage(0, cur);
    for (int t0 = 0; t0 < n_slots; t0 += KT) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (t0 + KT < n_slots) stage(t0 + KT, other);
      typedef __attribute__((address_space(3))) const f32x4 lds_f32x4;
      typedef __attribute__((address_space(3))) const float lds_f32;
#pragma unroll(D == 128 ? 1 : 2)                           // (head size 128: the unrolled body spills)
      for (int h2 = 0; h2 < 2; ++h2) {                     // 32 slots
        // (unrolled, h2 is a constant offset and both halves share their address registers)
        constexpr bool U = D < 128;
        const unsigned qn = cur + qnat + (U ? 0 : 32 * RK * h2), qt = cur + qtr + (U ? 0 : 32 * RK * h2);
        const unsigned dn = cur + dnat + (U ? 0 : 32 * RV * h2), dt0 = cur + dtr + (U ? 0 : 32 * RV * h2);
        const int hc = U ? h2 : 0;
        const unsigned st0 = cur + KT * (2 * RK + RV) + 16 * (8 * g + 32 * h2);   // [64] lse1, lse2, delta1, delta2; then [64] lam, ...
        bf16x8 pf[KB], dsf[KB][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          f32x4 s[KB][2], dp[KB];
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) s[kb][0] = s[kb][1] = dp[kb] = (f32x4){0.f, 0.f, 0.f, 0.f};
          da_pipe<AK, 2 * KS + ES>([&](int i) { return i < 2 * KS ? da_nat<RK>(qn, hc, half, i >> 1, (i & 1) * KT * RK) : da_nat<RV>(dn, hc, half, i - 2 * KS); },
                               [&](int i, bf16x8 x) {
#pragma unroll
                                 for (int kb = 0; kb < KB; ++kb) {
                                   if (i < 2 * KS) s[kb][i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, kf[kb][i & 1][i >> 1], s[kb][i & 1], 0, 0, 0);
                                   else dp[kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, vf[kb][i - 2 * KS], dp[kb], 0, 0, 0);
                                 }
                               });
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const unsigned at = st0 + 16 * (4 * half + r);
            const f32x4 st = *(lds_f32x4*)(size_t)at;
            const float lam = *(lds_f32*)(size_t)(at + 1024);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              const float p1 = __builtin_amdgcn_exp2f(s[kb][0][r] * scale2 - st[0]);
              const float p2 = __builtin_amdgcn_exp2f(s[kb][1][r] * scale2 - st[1]) * lam;
              // to bf16 as the products' operands, the maps' difference taken before: 2^-8 of each difference, of each dS
              pf[kb][4 * half + r] = (__bf16)(p1 - p2);
              dsf[kb][0][4 * half + r] = (__bf16)(p1 * (dp[kb][r] - st[2]));
              dsf[kb][1][4 * half + r] = (__bf16)(p2 * (st[3] - dp[kb][r]));
            }
          }
        }
        // dV^T += dO^T P, dKm^T += Qm^T dSm
        da_pipe<AK, ET + 2 * DT>([&](int i) { return i < ET ? da_tr<RV>(dt0, hc, i) : da_tr<RK>(qt, hc, (i - ET) >> 1, ((i - ET) & 1) * KT * RK); },
                             [&](int i, bf16x8 x) {
#pragma unroll
                               for (int kb = 0; kb < KB; ++kb) {
                                 if (i < ET) av[kb][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, pf[kb], av[kb][i], 0, 0, 0);
                                 else {
                                   f32x4& z = ak[kb][(i - ET) & 1][(i - ET) >> 1];
                                   z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, dsf[kb][(i - ET) & 1], z, 0, 0, 0);
                                 }
                               }
                             });
      }
      const unsigned sw = cur; cur = other; other = sw;
    }
  }
  const int k1 = da_again(k0), g1 = da_again(lane) >> 4;
  const float scale = n_slots > 0 ? *(const float*)(sb0 + 20) : 0.f;   // (the same of every slot: they see the same keys)
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int key = k1 + 16 * kb;
    if (key >= sp.Lk) continue;
    const bool vis = !a.mask || a.mask[b * a.mask_stride + key] != 0;
    // a masked key's gradients are exact zeros whatever its column held
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      unsigned short* op = a.dk + bq * a.dks[0] + (sp.k0 + key) * a.dks[1] + (2 * hk + m) * a.dks[2] + 4 * g1;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        u32x2 w = {0u, 0u};
        if (vis) {
          w[0] = bd_pack_bf16x2(ak[kb][m][dt][0] * scale, ak[kb][m][dt][1] * scale);
          w[1] = bd_pack_bf16x2(ak[kb][m][dt][2] * scale, ak[kb][m][dt][3] * scale);
        }
        *(u32x2*)(op + 16 * dt) = w;
      }
    }
    unsigned short* op = a.dv + bq * a.dvs[0] + (sp.k0 + key) * a.dvs[1] + hk * a.dvs[2] + 4 * g1;
#pragma unroll
    for (int dt = 0; dt < ET; ++dt) {
      u32x2 w = {0u, 0u};
      if (vis) {
        w[0] = bd_pack_bf16x2(av[kb][dt][0], av[kb][dt][1]);
        w[1] = bd_pack_bf16x2(av[kb][dt][2], av[kb][dt][3]);
      }
      *(u32x2*)(op + 16 * dt) = w;
    }
  }
}

// dlam [B, L, H] summed over the axes that lam was broadcast along (kept axes: kb, kl, kh), in a fixed order; one
// workgroup per kept value, eight loads of a thread in flight (a weight per head, 32 768 rows: 6 us; one load at a time 59)
template <typename T>
__global__ __launch_bounds__(1024) void da_dlam_kernel(const float* __restrict__ dlam, T* __restrict__ out, int B, int L, int H, int kb, int kl,
                                                       int kh) {
  __shared__ float part[16];
  const int nh = kh ? H : 1, nl = kl ? L : 1;
  const int h = blockIdx.x % nh, l = (blockIdx.x / nh) % nl, b = blockIdx.x / nh / nl;
  // the values summed: `rows` of them `step` apart, and, where the heads are summed too, H neighbours of each
  const float* p = dlam + ((long long)b * L + l) * H + h;
  long long rows = (kb ? 1ll : B) * (kl ? 1 : L), step = kl ? (long long)L * H : H, near = kh ? 1 : H;
  if (near > 1 && (step == H || rows == 1)) { rows *= near; step = near = 1; }
  const long long n = rows * near;
  float s = 0.f;
  for (long long i = threadIdx.x; i < n; i += 8 * 1024) {
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const long long k = i + 1024 * u;
      x[u] = k < n ? p[near == 1 ? k * step : k / near * step + k % near] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) s += x[u];
  }
  s = bd_wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.f;
    for (int w = 0; w < 16; ++w) s += part[w];
    if (sizeof(T) == 2) out[blockIdx.x] = (T)bd_f32_to_bf16(s);
    else ((float*)out)[blockIdx.x] = s;
  }
}

// ---------------------------------------------------------------------------------------------- host side
// Forward: blocks of 16 slots a wave holds, query groups of a workgroup (two waves each), waves of a SIMD. Measured, forward
// alone: head size 64, 16 x 1024 tokens x 3 heads: (1, 4, 4) 59 us, (2, 2, 2) 60, (2, 4, 2) 70, (1, 2, 4) 70; 256 x 128
// padded tokens 32.6, 34.1, 36.7, 43.7. Head size 128, 2 x 4096 x 8 over 4: (2, 4, 2) 391 us, (1, 4, 2) 492, (2, 2, 2) 558,
// (1, 2, 2) 722 (few slots a workgroup: the tiles' way into LDS paces it). Head size 32, 96 ragged sequences x 8: (2, 2, 4)
// 85 us, (1, 4, 6) 98, (1, 4, 5) 109, (1, 2, 6) 118, (2, 1, 4) 129, (1, 8, 4) 151.
template <int B_, int NQG_, int OCC_> struct DaFCfg { static constexpr int B = B_, NQG = NQG_, OCC = OCC_, SLOTS = 16 * B_ * NQG_; };
template <int D> struct DaFwd : DaFCfg<1, 4, 4> {};
template <> struct DaFwd<32> : DaFCfg<2, 2, 4> {};
template <> struct DaFwd<128> : DaFCfg<2, 4, 2> {};
constexpr int ROWS_NQG = 2, ROWS_SLOTS = 16 * ROWS_NQG;                         // few slots: 32, 4 waves of 16

// The forward of a call. Half of the large workgroup's slots or fewer: the workgroup of 32 (measured, this / the large one:
// 2 rows against 512 keys x 6 heads of 64 in 64 sequences 15.6 / 20.1 us, 32 rows 16.1 / 21.1, 64 rows 23.4 / 22.5; heads of
// 128, 32 rows 31.5 / 57.5, 64 rows 46.4 / 58.8). Split over the keys where the workgroups leave CUs without work, one a CU,
// if that gives a split enough key tiles: 2 for the workgroup of 32 (one row against 4096 keys, 4 heads of 64 over 4 key
// heads: 10.3 us, with 4 tiles 11.9, with 8 15.5), else 16 (1024 rows against 1024 keys, 8 heads of 64: 20.0 us unsplit,
// 28.5 with 8 tiles, 33.0 with 4; 128 rows against 4096 keys, 16 heads over 4: unsplit 62, split in four 30). 65 521 keys,
// 16 heads over 4, split / unsplit: 16 rows 37 / 927 us, 128 rows 150 / 937, 512 rows 561 / 944.
struct DaPlan { bool few; int per, n_blk, n_split; };

DaPlan da_plan(const bd_diff_attn_args& p) {
  const long long slots = (long long)p.Lq * (p.H / p.Hkv);
  const int large = p.head_dim == 128 ? DaFwd<128>::SLOTS : p.head_dim == 64 ? DaFwd<64>::SLOTS : DaFwd<32>::SLOTS;
  DaPlan r;
  r.few = 2 * slots <= large;
  r.per = r.few ? ROWS_SLOTS : large;
  r.n_blk = (int)((slots + r.per - 1) / r.per);
  const int most = (p.Lk + KT - 1) / KT / (r.few ? 2 : 16);
  long long n = 256 / ((long long)p.B * p.Hkv * r.n_blk);
  if (n > most) n = most;
  r.n_split = p.cu_seqlens || n < 1 ? 1 : n > JOIN_SPLITS ? JOIN_SPLITS : (int)n;
  return r;
}

int da_check(const bd_diff_attn_args& p, const char* what, DaArgs& a) {
  BD_REQUIRE(p.q && p.k && p.v && p.lam, "%s: null operand", what);
  BD_REQUIRE(p.B > 0 && p.Lq > 0 && p.Lk > 0 && p.H > 0 && p.Hkv > 0, "%s: empty shape", what);
  BD_REQUIRE(p.H % p.Hkv == 0, "%s: %d heads cannot share %d key heads evenly", what, p.H, p.Hkv);
  BD_REQUIRE(p.head_dim == 32 || p.head_dim == 64 || p.head_dim == 128, "%s: head_dim %d not in {32, 64, 128}", what, p.head_dim);
  BD_REQUIRE((long long)p.Lq * (p.H / p.Hkv) < (1ll << 30) && p.Lk < (1 << 30) && (long long)p.B * p.Hkv < (1ll << 24),
             "%s: too many rows or heads", what);
  BD_REQUIRE(!p.cu_seqlens || p.Lq == p.Lk, "%s: packed rows need Lq == Lk (the longest sequence)", what);
  BD_REQUIRE(!p.cu_seqlens || p.total_rows > 0, "%s: packed rows need total_rows", what);
  // (2^8 over the scale is how far a score may pass the running maximum: it has to be finite)
  BD_REQUIRE(p.scale >= 1e-30f && p.scale <= 1e30f, "%s: scale must lie within 1e-30 and 1e30", what);
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
  for (a.share_log = 0; (1 << a.share_log) < a.share;) ++a.share_log;
  a.share_mul = (unsigned)((1ull << (30 + a.share_log)) / a.share) + 1u;
  a.lam_f32 = p.lam_dtype == BD_DTYPE_F32; a.scale = p.scale; a.n_split = 1;
  a.small_strides = (long long)p.H * 32 * KT < (1ll << 31);
  for (int i = 1; i < 3; ++i)
    a.small_strides = a.small_strides && (unsigned long long)(p.q_stride[i] | p.k_stride[i] | p.v_stride[i] | p.dout_stride[i]) < (1ull << 24);
  a.lse = p.lse; a.maps = p.maps;
  return BD_OK;
}

template <int D>
int da_forward(const bd_diff_attn_args& p, DaArgs& a, hipStream_t s) {
  constexpr int LDS = 2 * KT * 8 * D;
  const long long slots = (long long)a.Lq * a.share;
  const int seqs = a.B + (a.cu ? 1 : 0);
  const DaPlan pl = da_plan(p);
  a.n_split = pl.n_split; a.n_blk = pl.n_blk; a.per = pl.per;
  const long long grid = da_grid((long long)a.n_blk * a.n_split, (long long)a.Hkv * seqs);
  BD_REQUIRE(grid < (1ll << 31), "bd_diff_attention_fwd: too many workgroups");
  if (a.n_split > 1) {
    a.part_ml = (float*)p.workspace;
    a.part = a.part_ml + (long long)a.n_blk * a.n_split * a.Hkv * a.B * 2 * a.per * 2;
  }
  typedef DaFwd<D> F;
  if (!pl.few) {
    BD_SET_MAX_LDS((da_fwd_kernel<D, F::B, F::NQG, F::OCC, false>), LDS);
    hipLaunchKernelGGL((da_fwd_kernel<D, F::B, F::NQG, F::OCC, false>), dim3((unsigned)grid), dim3(128 * F::NQG), LDS, s, a);
  } else if (a.n_split == 1) {
    BD_SET_MAX_LDS((da_fwd_kernel<D, 1, ROWS_NQG, 2, false>), LDS);
    hipLaunchKernelGGL((da_fwd_kernel<D, 1, ROWS_NQG, 2, false>), dim3((unsigned)grid), dim3(128 * ROWS_NQG), LDS, s, a);
  } else {
    BD_SET_MAX_LDS((da_fwd_kernel<D, 1, ROWS_NQG, 2, true>), LDS);
    hipLaunchKernelGGL((da_fwd_kernel<D, 1, ROWS_NQG, 2, true>), dim3((unsigned)grid), dim3(128 * ROWS_NQG), LDS, s, a);
  }
  if (a.n_split > 1) {
    constexpr int CB = 2 * D / JOIN_COLS;
    int lanes = 2;
    while (lanes < a.n_split) lanes *= 2;
    if (a.n_split <= JOIN_LANES)      // (16 splits of 512 slots x 4 key heads: 14.8 us, the other way 39.6)
      hipLaunchKernelGGL((da_join_few_kernel<D>), dim3((unsigned)((slots * lanes + 4 * JOIN_LANES - 1) / (4 * JOIN_LANES) * CB), a.Hkv, a.B), dim3(256),
                         0, s, a);
    else
      hipLaunchKernelGGL((da_join_kernel<D>), dim3((unsigned)(slots * CB), a.Hkv, a.B), dim3(256), 0, s, a);
  }
  return bd_check_launch("bd_diff_attention_fwd");
}

// Backward: blocks of 16 slots (dq) or keys (dkv) a wave holds, waves of a workgroup, waves of a SIMD. Measured: head size
// 64, 16 x 1024 x 3 heads: dq (2, 4, 2) 72 us, (1, 8, 4) 74, (1, 4, 4) 77, (2, 2, 2) 143; dkv (1, 4, 2) 79, (1, 8, 2) 94,
// (2, 4, 1) 116, (1, 4, 3) 308 (spills). Head size 128, 2 x 4096 x 8 over 4: dq (1, 8, 2) 435 us, (2, 4, 1) 497, (1, 4, 2)
// 1034; dkv (1, 8, 2) 713, (1, 4, 1) 819, (2, 4, 1) 872. Head size 32, 96 ragged x 8: dq (1, 4, 4) 86 us, (1, 4, 5) 95, (2,
// 4, 2) 97 (but 152 against 176 at 96 x 512), (1, 8, 5) 118; dkv (1, 4, 4) 94, (2, 2, 2) 95, (1, 4, 3) 98, (2, 4, 2) 112,
// (1, 8, 4) 115.
template <int B_, int NW_, int OCC_> struct DaCfg { static constexpr int B = B_, NW = NW_, OCC = OCC_; };
template <int D> struct DaBwd { typedef DaCfg<2, 4, 2> Q; typedef DaCfg<1, 4, 2> K; typedef DaCfg<1, 4, 3> QS; typedef DaCfg<1, 4, 3> QR; };
template <> struct DaBwd<32> { typedef DaCfg<1, 4, 4> Q; typedef DaCfg<1, 4, 4> K; typedef Q QS; typedef DaCfg<1, 4, 3> QR; };
template <> struct DaBwd<128> { typedef DaCfg<1, 8, 2> Q; typedef DaCfg<1, 8, 2> K; typedef DaCfg<1, 4, 2> QS; typedef Q QR; };

template <int D, typename C, bool SHORT>
void da_launch_dq(DaArgs& a, hipStream_t s, long long grid) {
  constexpr int LDS = 2 * KT * 8 * D;
  BD_SET_MAX_LDS((da_bwd_dq_kernel<D, C::B, C::NW, C::OCC, SHORT>), LDS);
  hipLaunchKernelGGL((da_bwd_dq_kernel<D, C::B, C::NW, C::OCC, SHORT>), dim3((unsigned)grid), dim3(64 * C::NW), LDS, s, a);
}

template <int D>
int da_backward(DaArgs& a, hipStream_t s) {
  constexpr int LDS_KV = 2 * KT * (8 * D + 32);
  typedef typename DaBwd<D>::Q Q;
  typedef typename DaBwd<D>::QS QS;
  typedef typename DaBwd<D>::QR QR;
  typedef typename DaBwd<D>::K K;
  const long long slots = (long long)a.Lq * a.share, groups = (long long)a.Hkv * (a.B + (a.cu ? 1 : 0));
  auto blocks = [](long long rows, int per) { return (rows + per - 1) / per; };
  // Workgroups for at most half of the CUs: smaller ones (dq, this / the large ones: 4096 tokens x 4 heads of 64 96 / 130
  // us, 1024 tokens 27 / 40; 4096 tokens x 4 heads of 128 146 / 180; 8192 x 3 heads of 128, three quarters of the CUs, 541 /
  // 374. dk / dv with half the keys a workgroup: 4096 x 4 heads of 128 338 / 306, 2048 x 7 of 64 78 / 64: not worth it)
  const bool small = 2 * (long long)a.Hkv * a.B * blocks(slots, 16 * Q::B * Q::NW) <= 256;
  // At most two key tiles: both stay in LDS, weights and dP in registers, the keys are walked once (this / the general form:
  // 256 x 128 padded tokens x 3 heads of 64 35.4 / 40.8 us, 8 x 128 8.9 / 12.0, 256 x 64 18.5 / 25.7; heads of 32, 256 x 128
  // 21.3 / 26.6)
  const bool keeps = D <= 64 && !a.maps && a.Lk <= 2 * KT;
  a.n_blk = (int)blocks(slots, keeps ? 16 * QR::B * QR::NW : small ? 16 * QS::B * QS::NW : 16 * Q::B * Q::NW);
  long long grid = da_grid(a.n_blk, groups);
  BD_REQUIRE(grid < (1ll << 31), "bd_diff_attention_bwd: too many workgroups");
  if (keeps) da_launch_dq<D, QR, D <= 64>(a, s, grid);
  else if (small) da_launch_dq<D, QS, false>(a, s, grid);
  else da_launch_dq<D, Q, false>(a, s, grid);
  if (!a.dk) return bd_check_launch("bd_diff_attention_bwd");
  a.n_blk = (int)blocks(a.Lk, 16 * K::B * K::NW);
  grid = da_grid(a.n_blk, groups);
  BD_REQUIRE(grid < (1ll << 31), "bd_diff_attention_bwd: too many workgroups");
  BD_SET_MAX_LDS((da_bwd_dkv_kernel<D, K::B, K::NW, K::OCC>), LDS_KV);
  hipLaunchKernelGGL((da_bwd_dkv_kernel<D, K::B, K::NW, K::OCC>), dim3((unsigned)grid), dim3(64 * K::NW), LDS_KV, s, a);
  return bd_check_launch("bd_diff_attention_bwd");
}

}  // namespace

extern "C" long long bd_diff_attention_workspace_bytes(const bd_diff_attn_args* p, int backward) {
  if (!p || p->B <= 0 || p->Lq <= 0 || p->Lk <= 0 || p->H <= 0 || p->Hkv <= 0 || p->H % p->Hkv) return -1;
  const long long rows = p->cu_seqlens ? p->total_rows : (long long)p->B * p->Lq;
  if (backward) return rows * p->H * 32;
  const DaPlan r = da_plan(*p);
  return r.n_split == 1 ? 0 : (long long)r.n_blk * r.n_split * p->Hkv * p->B * 2 * r.per * (2 + 2 * (long long)p->head_dim) * 4;
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
  BD_REQUIRE(p->dlam_dtype == BD_DTYPE_BF16 || p->dlam_dtype == BD_DTYPE_F32, "bd_diff_attention_bwd: dlam is neither bf16 nor fp32");
  BD_REQUIRE(p->dout && p->dlam && p->lse && !p->dk == !p->dv, "bd_diff_attention_bwd: null operand (dq may be, dk and dv together)");
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
  a.dlam = p->dlam; a.dlam_bf16 = p->dlam_dtype == BD_DTYPE_BF16;
  a.stats = (float*)p->workspace;
  bd_prof_scope prof(stream, (p->dk ? 28.0 : 12.0) * p->B * p->H * (double)p->Lq * p->Lk * p->head_dim, BD_PROF_ATTN_BWD);
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
  BD_REQUIRE(all < (1ll << 38) && kept < (1ll << 31), "bd_diff_attention_dlam: too many values");
  hipStream_t s = (hipStream_t)stream;
  const bool bf = out_dtype == BD_DTYPE_BF16;
  const dim3 grid((unsigned)kept);
  if (bf) hipLaunchKernelGGL(da_dlam_kernel<unsigned short>, grid, dim3(1024), 0, s, dlam, (unsigned short*)out, B, L, H, keep_b, keep_l, keep_h);
  else hipLaunchKernelGGL(da_dlam_kernel<float>, grid, dim3(1024), 0, s, dlam, (float*)out, B, L, H, keep_b, keep_l, keep_h);
  return bd_check_launch("bd_diff_attention_dlam");
}
