// Rotary positions (gfx950): pairs of a head's values turned by an angle that grows with the token's position.
//
//   y_a = x_a cos(phi) - x_b sin(phi),  y_b = x_a sin(phi) + x_b cos(phi),  phi = position * frequency_i
//
// for the rd / 2 pairs (a, b) of a head: (i, i + rd / 2) in the half layout, (2 i, 2 i + 1) interleaved. The values
// behind the first rd of a head are copied (left alone in place). cos and sin come from a table of the caller's
// [table_rows, rd / 2, 2] in fp32, so that far positions keep angles evaluated in 64 bits and any rule that stretches
// or scales them is the table's. The backward pass is the same kernel with the sine's sign turned (the transpose).
//
// Bound by memory: every value is read and written once. A thread turns one unit of 2 x 16 bytes (8 bf16 or 4 fp32
// pairs) of up to four heads: the unit's table entries stay in its registers, neighbouring lanes take neighbouring
// units and heads of one token (whole lines, the same table row), and the loads of all its heads are in flight together.
// Measured: 30 011 tokens x 20 heads of 128 in fp32, half of each turned, 115 us (614 MB read and written: 5.3 TB/s; a large
// copy runs at 4.9); 256 x 128 tokens x 6 heads of 128 in bf16 18.2 us (101 MB: 5.5 TB/s, part of it from the last-level
// cache); 64 x 2 tokens x 24 heads of 64 3.5 us, a launch's latency.
#include "bd_common.h"
#include "bd_prof.h"
#include "bidiff.h"

namespace {

struct RotArgs {
  bd_rotary_tensor t[2];
  const float* table;
  const long long* positions;
  long long pos_stride;
  int table_rows, B, L, D, rd, heads0, heads, slots, units, tail, items;
  int interleaved, inverse;
};

template <typename T> struct RotVec;
template <> struct RotVec<unsigned short> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const unsigned short* p, float (&v)[8]) {
    const u32x4 w = *(const u32x4*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ void store(unsigned short* p, const float (&v)[8]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = bd_pack_bf16x2(v[2 * i], v[2 * i + 1]);
    *(u32x4*)p = w;
  }
};
template <> struct RotVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
    const f32x4 w = *(const f32x4*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = w[i];
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    f32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = v[i];
    *(f32x4*)p = w;
  }
};
__device__ __forceinline__ float rot_get(const unsigned short* p) { return bd_bf16_to_f32(*p); }
__device__ __forceinline__ float rot_get(const float* p) { return *p; }
__device__ __forceinline__ void rot_put(unsigned short* p, float v) { *p = bd_f32_to_bf16(v); }
__device__ __forceinline__ void rot_put(float* p, float v) { *p = v; }

// the fused steps are written out: every kernel below then rounds alike, whichever of them a call takes
__device__ __forceinline__ void rot_pair(float xa, float xb, float cs, float sn, float& ya, float& yb) {
  ya = __builtin_fmaf(xa, cs, -(xb * sn));
  yb = __builtin_fmaf(xa, sn, xb * cs);
}

__device__ __forceinline__ long long rot_position(const RotArgs& a, int b, int l) {
  return a.positions ? a.positions[(long long)b * a.pos_stride + l] : (long long)l;
}

// item = ((token * slots) + slot) * (units + tail) + unit; slot s takes the heads s, s + slots, ... (at most G)
template <typename T, int G>
__global__ __launch_bounds__(256) void rotary_vec_kernel(RotArgs a) {
  constexpr int N = RotVec<T>::N;
  const int item = blockIdx.x * 256 + threadIdx.x;
  if (item >= a.items) return;
  const int per = a.units + a.tail;
  const int u = item % per, ts = item / per;
  const int slot = ts % a.slots, tok = ts / a.slots;
  const int b = tok / a.L, l = tok - b * a.L;
  const T* src[G];
  T* dst[G];
  int n = 0;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int h = slot + i * a.slots;
    if (h >= a.heads) break;
    const int w = h >= a.heads0;
    const bd_rotary_tensor& t = a.t[w];
    const int hh = w ? h - a.heads0 : h;
    src[i] = (const T*)t.src + (b * t.src_stride[0] + l * t.src_stride[1] + hh * t.src_stride[2]);
    dst[i] = (T*)t.dst + (b * t.dst_stride[0] + l * t.dst_stride[1] + hh * t.dst_stride[2]);
    n = i + 1;
  }
  if (u >= a.units) {                                    // behind the rotated part: copied
    const int e = a.rd + (u - a.units) * N;
#pragma unroll
    for (int i = 0; i < G; ++i)
      if (i < n) *(u32x4*)(dst[i] + e) = *(const u32x4*)(src[i] + e);
    return;
  }
  const int ea = a.interleaved ? 2 * N * u : N * u, eb = a.interleaved ? ea + N : ea + a.rd / 2;
  float xa[G][N], xb[G][N];
#pragma unroll
  for (int i = 0; i < G; ++i)
    if (i < n) { RotVec<T>::load(src[i] + ea, xa[i]); RotVec<T>::load(src[i] + eb, xb[i]); }
  float cs[N], sn[N];
  const long long pos = rot_position(a, b, l);
  if (pos >= 0 && pos < a.table_rows) {
    const float* tp = a.table + (size_t)pos * a.rd + 2 * N * u;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const f32x4 w = *(const f32x4*)(tp + 4 * i);
      cs[2 * i] = w[0]; sn[2 * i] = w[1]; cs[2 * i + 1] = w[2]; sn[2 * i + 1] = w[3];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) cs[i] = sn[i] = __uint_as_float(0x7fc00000u);
  }
  if (a.inverse) {
#pragma unroll
    for (int i = 0; i < N; ++i) sn[i] = -sn[i];
  }
#pragma unroll
  for (int i = 0; i < G; ++i) {
    if (i >= n) break;
    float ya[N], yb[N];
    if (a.interleaved) {                                 // pairs (2 j, 2 j + 1) of the 2 N values xa | xb
#pragma unroll
      for (int j = 0; j < N / 2; ++j) {
        rot_pair(xa[i][2 * j], xa[i][2 * j + 1], cs[j], sn[j], ya[2 * j], ya[2 * j + 1]);
        rot_pair(xb[i][2 * j], xb[i][2 * j + 1], cs[N / 2 + j], sn[N / 2 + j], yb[2 * j], yb[2 * j + 1]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) rot_pair(xa[i][j], xb[i][j], cs[j], sn[j], ya[j], yb[j]);
    }
    RotVec<T>::store(dst[i] + ea, ya);
    RotVec<T>::store(dst[i] + eb, yb);
  }
}

// any even rd, any strides and alignment: one pair (or one copied value) of one head per thread
template <typename T>
__global__ __launch_bounds__(256) void rotary_any_kernel(RotArgs a) {
  const int item = blockIdx.x * 256 + threadIdx.x;
  if (item >= a.items) return;
  const int per = a.units + a.tail;
  const int u = item % per, th = item / per;
  const int h = th % a.heads, tok = th / a.heads;
  const int b = tok / a.L, l = tok - b * a.L;
  const int w = h >= a.heads0;
  const bd_rotary_tensor& t = a.t[w];
  const int hh = w ? h - a.heads0 : h;
  const T* src = (const T*)t.src + (b * t.src_stride[0] + l * t.src_stride[1] + hh * t.src_stride[2]);
  T* dst = (T*)t.dst + (b * t.dst_stride[0] + l * t.dst_stride[1] + hh * t.dst_stride[2]);
  if (u >= a.units) {
    dst[a.rd + u - a.units] = src[a.rd + u - a.units];
    return;
  }
  const int ea = a.interleaved ? 2 * u : u, eb = a.interleaved ? ea + 1 : ea + a.rd / 2;
  const long long pos = rot_position(a, b, l);
  float cs = __uint_as_float(0x7fc00000u), sn = cs;
  if (pos >= 0 && pos < a.table_rows) {
    cs = a.table[(size_t)pos * a.rd + 2 * u];
    sn = a.table[(size_t)pos * a.rd + 2 * u + 1];
  }
  if (a.inverse) sn = -sn;
  const float xa = rot_get(src + ea), xb = rot_get(src + eb);
  float ya, yb;
  rot_pair(xa, xb, cs, sn, ya, yb);
  rot_put(dst + ea, ya);
  rot_put(dst + eb, yb);
}

template <typename T>
int rotary_launch(RotArgs& a, bool vec, bool in_place, hipStream_t s) {
  constexpr int N = RotVec<T>::N;
  const long long tokens = (long long)a.B * a.L;
  long long items;
  if (vec) {
    a.units = a.rd / (2 * N);
    a.tail = in_place ? 0 : (a.D - a.rd) / N;
    // four heads a thread where that still leaves more threads than the card holds at once (256 CUs x 2048). Measured, one head
    // a thread / four: the fp32 case above 117.5 / 116.2 us (the 2 it takes: 115.5), 64 x 2 tokens x 24 heads 3.5 / 5.1
    const int per = a.units + a.tail;
    int g = 1;
    while (g < 4 && tokens * ((a.heads + 2 * g - 1) / (2 * g)) * per >= 256 * 2048) g *= 2;
    a.slots = (a.heads + g - 1) / g;
    items = tokens * a.slots * per;
    BD_REQUIRE(items < (1ll << 31) - 256, "bd_rotary: too many values in one call");
    a.items = (int)items;
    const dim3 grid((unsigned)((items + 255) / 256));
    if (g == 1) hipLaunchKernelGGL((rotary_vec_kernel<T, 1>), grid, dim3(256), 0, s, a);
    else if (g == 2) hipLaunchKernelGGL((rotary_vec_kernel<T, 2>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rotary_vec_kernel<T, 4>), grid, dim3(256), 0, s, a);
  } else {
    a.units = a.rd / 2;
    a.tail = in_place ? 0 : a.D - a.rd;
    items = tokens * a.heads * (a.units + a.tail);
    BD_REQUIRE(items < (1ll << 31) - 256, "bd_rotary: too many values in one call");
    a.items = (int)items;
    hipLaunchKernelGGL((rotary_any_kernel<T>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, a);
  }
  return bd_check_launch("bd_rotary");
}

}  // namespace

extern "C" int bd_rotary(const bd_rotary_tensor* tensors, int n_tensors, const float* table, int table_rows,
                         const long long* positions, long long position_stride, int B, int L, int head_dim, int rotary_dim,
                         int interleaved, int inverse, int dtype, void* stream) {
  BD_REQUIRE(tensors && table && (n_tensors == 1 || n_tensors == 2), "bd_rotary: null operand or a tensor count that is not 1 or 2");
  BD_REQUIRE(B > 0 && L > 0 && table_rows > 0, "bd_rotary: empty shape");
  BD_REQUIRE((long long)B * L < (1ll << 31), "bd_rotary: too many tokens");
  BD_REQUIRE(head_dim > 0 && rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
             "bd_rotary: rotary_dim %d must be even and within the head size %d", rotary_dim, head_dim);
  BD_REQUIRE(dtype == BD_DTYPE_BF16 || dtype == BD_DTYPE_F32, "bd_rotary: dtype %d is neither bf16 nor fp32", dtype);
  RotArgs a;
  a.table = table; a.positions = positions; a.pos_stride = position_stride; a.table_rows = table_rows;
  a.B = B; a.L = L; a.D = head_dim; a.rd = rotary_dim;
  a.interleaved = interleaved != 0; a.inverse = inverse != 0;
  a.heads0 = tensors[0].n_heads; a.heads = 0;
  const int N = dtype == BD_DTYPE_BF16 ? 8 : 4;
  bool vec = rotary_dim % (2 * N) == 0 && head_dim % N == 0 && ((uintptr_t)table & 15) == 0;
  bool in_place = true;
  for (int i = 0; i < n_tensors; ++i) {
    const bd_rotary_tensor& t = tensors[i];
    BD_REQUIRE(t.src && t.dst && t.n_heads > 0, "bd_rotary: null tensor or no heads");
    a.t[i] = t;
    a.heads += t.n_heads;
    vec = vec && (((uintptr_t)t.src | (uintptr_t)t.dst) & 15) == 0;
    for (int k = 0; k < 3; ++k) vec = vec && t.src_stride[k] % N == 0 && t.dst_stride[k] % N == 0;
    in_place = in_place && t.src == t.dst;
    for (int k = 0; k < 3; ++k)
      BD_REQUIRE(t.src != t.dst || t.src_stride[k] == t.dst_stride[k], "bd_rotary: in place, source and destination need the same strides");
  }
  if (n_tensors == 1) a.t[1] = a.t[0];
  bd_prof_scope prof(stream, 2.0 * B * L * (double)a.heads * head_dim * (dtype == BD_DTYPE_BF16 ? 2 : 4), BD_PROF_EMBED);
  return dtype == BD_DTYPE_BF16 ? rotary_launch<unsigned short>(a, vec, in_place, (hipStream_t)stream)
                                : rotary_launch<float>(a, vec, in_place, (hipStream_t)stream);
}
