// The 4-bit KV cache: rows are quantised as they are written (tb200_kv4_append) and turned back into 16-bit rows
// (tb200_kv4_read).  A group is 64 consecutive values x of a row; with lo = min x and s = (max x - min x) / 15 it is
// held as the codes c = round((x - lo) / s) and the pair (s, lo) in the cache's 16-bit type, and stands for lo + c s.
// 64 values take 32 + 4 bytes: 4.5 bits per value.
//
// Bound: HBM (one row of D = 128 moves 256 + 72 bytes) and the instructions per value.  Reading 8 sequences of 1 to 8192
// rows, 8 heads of 128, fp16: 26.1 us, 146 MB at 85 % of the copy bandwidth.  Appending 8 prompts of 1 to 4093 rows, bf16,
// and reading them back: 40.9 us, 179 MB at 67 %; the append alone 24.5 us, 90 MB at 56 %, an instruction issued in two thirds of
// the cycles.
#include "common.cuh"
#include "internal.h"
#include "kv4.cuh"

namespace tb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 2;   // rows of a thread: eight 16-byte loads in flight

struct RowsParams {
  const int32_t* start;
  const int32_t* n_rows;
  int start_all, rows, heads, cache_len;
  long long n_bh;           // batch * heads
  long long units;          // of rows, times n_bh
  uint8_t* x[2];            // k, v
  long long stride[2][3];   // elements: batch, head, row
  uint8_t* codes[2];
  uint8_t* meta[2];
  // SEEN: n_rows are the sequences' lengths, rows the positions of the 16-bit copy
  const int32_t* q_rows;
  int q_rows_max, window, sinks, packed_head;
  const float4* head_factor;
};

template <typename T> struct Bits;   // a 16-bit value and its raw bits
template <> struct Bits<__half> {
  static __device__ __forceinline__ float f(uint32_t u) { return __half2float(__ushort_as_half(static_cast<unsigned short>(u))); }
  static __device__ __forceinline__ uint32_t rn(float v) { return __half_as_ushort(__float2half_rn(v)); }
};
template <> struct Bits<__nv_bfloat16> {
  static __device__ __forceinline__ float f(uint32_t u) { return __uint_as_float(u << 16); }
  static __device__ __forceinline__ uint32_t rn(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
};

// Two 16-bit values at once: minimum and maximum (a NaN wins).
template <typename T> __device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b);
template <typename T> __device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t min2_nan<__half>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <> __device__ __forceinline__ uint32_t min2_nan<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <> __device__ __forceinline__ uint32_t max2_nan<__half>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <> __device__ __forceinline__ uint32_t max2_nan<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// x / 15 correctly rounded: the Newton step of encode8, with 1/15 rounded by the compiler; where the remainder would leave
// fp32's normal range, a division.
__device__ __forceinline__ float fifteenth(float x) {
  constexpr float kInv = 1.f / 15.f;
  const float q = __fmul_rn(x, kInv);
  const float r = __fmaf_rn(__fmaf_rn(q, -15.f, x), kInv, q);
  return x < 1e-30f ? __fdiv_rn(x, 15.f) : r;
}
// Below this scale encode8 divides.  fp16, 2^-19: s is rounded so coarsely (steps of 2^-24) that a quotient may pass 15.5.
// bf16, 2^-120: the Newton step's remainder may need digits below fp32's smallest.
template <typename T> struct SmallScale;
template <> struct SmallScale<__half> { static constexpr float value = 1.9073486328125e-06f; };
template <> struct SmallScale<__nv_bfloat16> { static constexpr float value = 7.52316385e-37f; };

// Codes of eight values of a group: round(t / s), halves to even, with t = x - lo rounded to fp32.  bf16 values lie on few
// places, so a quotient is exactly k + 1/2 in about one group of eight out of twenty, and it has to come out as just that: the
// approximate quotient q0 = t inv is followed by one Newton step, q = q0 + (t - q0 s) inv with the remainder exact in a fused
// multiply-add (P. Markstein, IBM J. Res. Dev. 34, 1990), which is t / s correctly rounded.  Adding 1.5 * 2^23 rounds q to a
// whole number and leaves the code in the sum's low bits.  (An x that is tiny beside lo is gone from t: where -lo / s is
// k + 1/2, its code is the even one, whatever its sign.  Both codes are as far from x, to 2^-19 s.)
// (Approximate quotients re-examined in 64 bits wherever one lay next to a border took twice as long.)
template <typename T>
__device__ __forceinline__ uint32_t encode8(const uint32_t (&w)[4], float lo, float s) {
  constexpr float kMagic = 12582912.f;
  const float inv = __fdividef(1.f, s);
  const float2 nlo = make_float2(-lo, -lo), inv2 = make_float2(inv, inv), ns = make_float2(-s, -s), magic = make_float2(kMagic, kMagic);
  uint32_t word = 0;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    const float2 t = __fadd2_rn(Pack2<T>::unpack(w[i]), nlo);
    const float2 q0 = __fmul2_rn(t, inv2);
    const float2 r = __fadd2_rn(__ffma2_rn(__ffma2_rn(q0, ns, t), inv2, q0), magic);
    word = word * 16 + __float_as_uint(r.y);
    word = word * 16 + __float_as_uint(r.x);
  }
  // every sum carries the bits of 1.5 * 2^23 along: taken out once for all eight
  constexpr uint32_t kBits = 0x4b400000u;
  constexpr uint32_t kCarry = kBits * 0x11111111u;
  word -= kCarry;
  if (!(s >= SmallScale<T>::value)) {   // 0, NaN or small
    word = 0;
    if (s > 0.f) {
#pragma unroll 1
      for (int i = 7; i >= 0; --i) {
        const float2 x2 = Pack2<T>::unpack(i < 2 ? w[0] : i < 4 ? w[1] : i < 6 ? w[2] : w[3]);
        word = word * 16 + static_cast<uint32_t>(fminf(rintf(__fdiv_rn(((i & 1) ? x2.y : x2.x) - lo, s)), 15.f));
      }
    }
  }
  return word;
}

// Four lanes share a group: lane l holds the eight values from 8 l on and the eight from 32 + 8 l on, so that every access of
// the four is one stretch of 64 bytes and what is done once per group costs half of what eight lanes spend on it.
// A unit is kUnitRows rows of one (sequence, head), k and v; units next to one another are of different sequences, so that
// short sequences leave no CTA without work.
template <int D> struct RowsShape {
  static constexpr int kLanes = D / 16;                // lanes per row
  static constexpr int kRows = kThreads / kLanes;      // rows side by side
  static constexpr int kUnitRows = kRows * kPerThread;
};
struct Unit {
  long long bh;
  int b, h, row0, n, start;
};
__device__ __forceinline__ Unit find_unit(const RowsParams& p, long long u, int unit_rows) {
  Unit x;
  int rb;
  if (p.units < (1LL << 31)) {   // (64-bit divisions for every unit: 3 % of the time of long prompts)
    const uint32_t u32 = static_cast<uint32_t>(u), n_bh = static_cast<uint32_t>(p.n_bh), heads = static_cast<uint32_t>(p.heads);
    const uint32_t r = u32 / n_bh, bh = u32 - r * n_bh, b = bh / heads;
    rb = static_cast<int>(r);
    x.bh = bh;
    x.b = static_cast<int>(b);
    x.h = static_cast<int>(bh - b * heads);
  } else {
    const long long r = u / p.n_bh;
    rb = static_cast<int>(r);
    x.bh = u - r * p.n_bh;
    x.b = static_cast<int>(x.bh / p.heads);
    x.h = static_cast<int>(x.bh - static_cast<long long>(x.b) * p.heads);
  }
  x.row0 = rb * unit_rows;
  x.n = p.n_rows ? min(p.n_rows[x.b], p.rows) : p.rows;
  x.start = p.start ? p.start[x.b] : p.start_all;
  return x;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 4) kv4_append_kernel(const __grid_constant__ RowsParams p) {
  using S = RowsShape<D>;
  const int r_in = threadIdx.x / S::kLanes, lane = threadIdx.x % S::kLanes;
  const int chunk = (lane >> 2) * 8 + (lane & 3);   // of eight values; the other one is four further on
  for (long long u = blockIdx.x; u < p.units; u += gridDim.x) {
    const Unit x = find_unit(p, u, S::kUnitRows);
    if (x.row0 >= x.n) continue;   // the whole CTA
    uint4 raw[kPerThread][2][2];
    bool live[kPerThread];
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int row = x.row0 + k * S::kRows + r_in;
      const long long pos = static_cast<long long>(x.start) + row;
      live[k] = row < x.n && pos >= 0 && pos < p.cache_len;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        raw[k][w][0] = raw[k][w][1] = make_uint4(0u, 0u, 0u, 0u);
        if (live[k]) {
          const uint4* src = reinterpret_cast<const uint4*>(p.x[w] + 2 * (x.b * p.stride[w][0] + x.h * p.stride[w][1] + row * p.stride[w][2])) + chunk;
          raw[k][w][0] = __ldcs(src);
          raw[k][w][1] = __ldcs(src + 4);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      if (!__any_sync(0xffffffffu, live[k])) continue;   // a warp's rows of which none is meant
      const long long crow = x.bh * p.cache_len + x.start + x.row0 + k * S::kRows + r_in;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t v[2][4] = {{raw[k][w][0].x, raw[k][w][0].y, raw[k][w][0].z, raw[k][w][0].w},
                                  {raw[k][w][1].x, raw[k][w][1].y, raw[k][w][1].z, raw[k][w][1].w}};
        // minimum, and minus the maximum (from here on a minimum, too) side by side in one register
        uint32_t lo2 = v[0][0], hi2 = v[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) {
          lo2 = min2_nan<T>(lo2, v[i >> 2][i & 3]);
          hi2 = max2_nan<T>(hi2, v[i >> 2][i & 3]);
        }
        hi2 ^= 0x80008000u;
        uint32_t both = min2_nan<T>(__byte_perm(lo2, hi2, 0x5410), __byte_perm(lo2, hi2, 0x7632));
        both = min2_nan<T>(both, __shfl_xor_sync(0xffffffffu, both, 1));
        both = min2_nan<T>(both, __shfl_xor_sync(0xffffffffu, both, 2));
        const float2 f = Pack2<T>::unpack(both);
        const float lo = f.x, range = __fsub_rn(-f.y, f.x);
        const bool odd = !(range < INFINITY);    // an infinity or a NaN among the 64, or a range past fp32
        const uint32_t sb = odd ? 0x7fffu : Bits<T>::rn(fifteenth(range));
        const uint32_t lb = odd ? 0x7fffu : (both & 0xffffu);
        const float s = odd ? 0.f : Bits<T>::f(sb);
        const uint32_t word0 = encode8<T>(v[0], lo, s), word1 = encode8<T>(v[1], lo, s);
        if (live[k]) {
          uint32_t* c = reinterpret_cast<uint32_t*>(p.codes[w] + crow * (D / 2)) + chunk;
          c[0] = word0;
          c[4] = word1;
          if ((lane & 3) == 0) *reinterpret_cast<uint32_t*>(p.meta[w] + (crow * (D / 64) + (lane >> 2)) * 4) = sb | (lb << 16);
        }
      }
    }
  }
}

// The positions some query row of sequence b sees: [low, n) and those below few.  In the copy, places below `head` are those
// positions, places from there on to `places` are positions `off` further on.
struct SeenRows {
  int n, low, few, head, off, places;
};
__device__ __forceinline__ SeenRows seen_rows(const RowsParams& p, int b) {
  const int r = p.q_rows ? max(0, min(p.q_rows[b], p.q_rows_max)) : p.q_rows_max;
  SeenRows s;
  s.n = max(0, min(p.n_rows[b], p.cache_len));
  s.low = r == 0 ? s.n : p.window > 0 ? s.n - r - p.window + 1 : 0;
  s.few = r > 0 ? p.sinks : 0;
  const bool packed = p.packed_head >= 0 && s.low > p.sinks;   // (as the attention kernel has it)
  s.head = packed ? p.packed_head : 0;
  s.off = packed ? s.low - s.head : 0;
  s.places = s.n - s.off;
  return s;
}

// Eight codes as fp16 values of (lo + c s) * down.
__device__ __forceinline__ uint4 decode8_scaled(uint32_t word, uint32_t meta, float down) {
  const float2 sl = Pack2<__nv_bfloat16>::unpack(meta);
  const float s = sl.x * down, lo = sl.y * down;
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = Pack2<__half>::pack(fmaf(static_cast<float>((word >> (8 * i)) & 15u), s, lo), fmaf(static_cast<float>((word >> (8 * i + 4)) & 15u), s, lo));
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// A power of two that brings `top`, or 2^(least - 127) where that is more, to [2^to, 2^(to + 1)), and its inverse; least > to.
__device__ __forceinline__ float2 power_for(float top, int to, int least) {
  const int ex = max(static_cast<int>(__float_as_uint(top) >> 23), least);
  return make_float2(__uint_as_float(static_cast<uint32_t>(254 + to - ex) << 23), __uint_as_float(static_cast<uint32_t>(ex - to) << 23));
}

// bf16 prompts on a 4-bit cache: the powers of two.  CTAs (i < kv heads, b): the largest magnitude among the seen rows of one
// (sequence, kv head) of K and of V, from s and lo alone; the CTAs behind them: rows of q, a warp each.  Infinities and NaN do
// not count.
struct FactorParams {
  RowsParams rows;
  int batch, q_heads;
  const uint8_t* q;
  long long q_stride[3];
  uint8_t* q16;
  float* q_factor;
  float4* head_factor;
};
constexpr int kFactorThreads = 1024;
template <int D>
__global__ void __launch_bounds__(kFactorThreads) kv4_factors_kernel(const __grid_constant__ FactorParams f) {
  const RowsParams& p = f.rows;
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float red[2][kFactorThreads / 32];
  for (int b = blockIdx.y; b < f.batch; b += gridDim.y) {
    if (blockIdx.x < p.heads) {
      const long long bh = static_cast<long long>(b) * p.heads + blockIdx.x;
      const SeenRows seen = seen_rows(p, b);
      const int n = seen.n, low = max(seen.low, 0), few = min(seen.few, low);
      float top[2] = {0.f, 0.f};
#pragma unroll 4
      for (int i = threadIdx.x; i < few + n - low; i += kFactorThreads) {
        const long long crow = bh * p.cache_len + (i < few ? i : i - few + low);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t u[D / 64];
          if constexpr (D == 128) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p.meta[w]) + crow);
            u[0] = v.x; u[1] = v.y;
          } else {
            u[0] = __ldg(reinterpret_cast<const uint32_t*>(p.meta[w]) + crow);
          }
#pragma unroll
          for (int g = 0; g < D / 64; ++g) {
            const float2 sl = Pack2<__nv_bfloat16>::unpack(u[g]);
            const float x = fmaxf(fabsf(sl.y), fabsf(fmaf(15.f, sl.x, sl.y)));   // (s is rounded: lo + 15 s may pass fp32's range)
            if (sl.x < INFINITY && fabsf(sl.y) < INFINITY) top[w] = fmaxf(top[w], fminf(x, 3.402823466e38f));
          }
        }
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], d));
        if (lane == 0) red[w][warp] = top[w];
      }
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          top[w] = red[w][lane];
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], d));
        }
        // below 2^15: fp16 ends at 65504.  V's inverse is divided by a sum of up to 2^39 before it meets the output: above 2^-102
        const float2 k = power_for(top[0], 14, 16), v = power_for(top[1], 14, 40);
        if (lane == 0) f.head_factor[bh] = make_float4(k.x, k.y, v.x, v.y);
      }
      __syncthreads();
      continue;
    }
    constexpr int V = D / 32;   // columns per lane
    const int rows = f.q_heads * p.q_rows_max, stride = (gridDim.x - p.heads) * (kFactorThreads / 32);
    const int live = p.q_rows ? p.q_rows[b] : p.q_rows_max;
    for (int row = (blockIdx.x - p.heads) * (kFactorThreads / 32) + warp; row < rows; row += stride) {
      const int h = row / p.q_rows_max, i = row - h * p.q_rows_max;
      if (i >= live) continue;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(f.q + 2 * (b * f.q_stride[0] + h * f.q_stride[1] + i * f.q_stride[2])) + lane * (V / 2);
      float2 x[V / 2];
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        x[e] = Pack2<__nv_bfloat16>::unpack(src[e]);
        const float m = fmaxf(fabsf(x[e].x), fabsf(x[e].y));
        top = fmaxf(top, m < INFINITY ? m : 0.f);
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float2 pw = power_for(top, 14, 16);
      const long long out = static_cast<long long>(b) * rows + row;
      uint32_t* dst = reinterpret_cast<uint32_t*>(f.q16 + out * D * 2) + lane * (V / 2);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) dst[e] = Pack2<__half>::pack(x[e].x * pw.x, x[e].y * pw.x);
      if (lane == 0) f.q_factor[out] = pw.y;
    }
  }
}

// SEEN: only the positions that some query row of the sequence sees (a prompt's attention reads the 16-bit rows next), bf16 as
// scaled fp16.
template <typename T, int D, bool SEEN>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const __grid_constant__ RowsParams p) {
  using S = RowsShape<D>;
  if constexpr (SEEN) {
    pdl_launch_dependents();
    pdl_wait();   // the factors
  }
  const int r_in = threadIdx.x / S::kLanes, lane = threadIdx.x % S::kLanes;
  const int chunk = (lane >> 2) * 8 + (lane & 3);
  for (long long u = blockIdx.x; u < p.units; u += gridDim.x) {
    Unit x = find_unit(p, u, S::kUnitRows);
    SeenRows seen;
    if constexpr (SEEN) {
      seen = seen_rows(p, x.b);
      x.n = seen.places;
    }
    if (x.row0 >= x.n) continue;
    float down[2] = {1.f, 1.f};
    if constexpr (SEEN) {
      if constexpr (IsBf16<T>::value) {
        const float4 f = __ldcg(p.head_factor + x.bh);
        down[0] = f.x;
        down[1] = f.z;
      }
    }
    uint32_t word[kPerThread][2][2], m[kPerThread][2];
    bool live[kPerThread];
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int row = x.row0 + k * S::kRows + r_in;
      long long pos = static_cast<long long>(x.start) + row;
      live[k] = row < x.n && pos >= 0 && pos < p.cache_len;
      if constexpr (SEEN) {
        pos = row < seen.head ? row : row + seen.off;
        live[k] = row < x.n && (row < seen.few || (row >= seen.head && pos >= seen.low));
      }
      if (!live[k]) continue;
      const long long crow = x.bh * p.cache_len + pos;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t* c = reinterpret_cast<const uint32_t*>(p.codes[w] + crow * (D / 2)) + chunk;
        word[k][w][0] = __ldcs(c);
        word[k][w][1] = __ldcs(c + 4);
        m[k][w] = __ldcs(reinterpret_cast<const uint32_t*>(p.meta[w] + (crow * (D / 64) + (lane >> 2)) * 4));
      }
    }
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      if (!live[k]) continue;
      const long long row = x.row0 + k * S::kRows + r_in;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint4* dst = reinterpret_cast<uint4*>(p.x[w] + 2 * (x.b * p.stride[w][0] + x.h * p.stride[w][1] + row * p.stride[w][2])) + chunk;
        if constexpr (SEEN && IsBf16<T>::value) {
          dst[0] = decode8_scaled(word[k][w][0], m[k][w], down[w]);
          dst[4] = decode8_scaled(word[k][w][1], m[k][w], down[w]);
        } else {
          dst[0] = Kv4Decode<T>::decode8(word[k][w][0], m[k][w]);
          dst[4] = Kv4Decode<T>::decode8(word[k][w][1], m[k][w]);
        }
      }
    }
  }
}

}  // namespace

int check_strides(const int64_t (&st)[3], const int64_t (&ext)[3], int head_dim, bool written) {
  int64_t s[3], e[3];
  int n = 0;
  for (int i = 0; i < 3; ++i) {
    if (ext[i] <= 1) continue;
    if (st[i] < head_dim || (st[i] & 7) || st[i] >= (1LL << 39)) return TB200_ERR_INVALID;
    int j = n++;
    for (; j > 0 && s[j - 1] > st[i]; --j) { s[j] = s[j - 1]; e[j] = e[j - 1]; }
    s[j] = st[i];
    e[j] = ext[i];
  }
  int64_t reach = head_dim;   // elements from the first to behind the last of the axes so far
  for (int i = 0; i < n; ++i) {
    if (written && s[i] < reach) return TB200_ERR_INVALID;
    reach += s[i] * (e[i] - 1);
  }
  return TB200_OK;
}

namespace {

int check_rows(const tb200_kv4_rows_args* a) {
  if (a == nullptr) return TB200_ERR_INVALID;
  if (a->dtype != TB200_BF16 && a->dtype != TB200_F16) return TB200_ERR_UNSUPPORTED;
  if (a->head_dim != 64 && a->head_dim != 128) return TB200_ERR_UNSUPPORTED;
  if (a->batch < 0 || a->rows < 0 || a->n_kv_heads < 1 || a->cache_len < 0 || (a->cache_len & 3) || a->reserved != 0) return TB200_ERR_INVALID;
  if (a->batch > kMaxExtent || a->rows > kMaxExtent || a->n_kv_heads > kMaxExtent || a->cache_len > kMaxExtent) return TB200_ERR_INVALID;
  if (a->batch == 0 || a->rows == 0 || a->cache_len == 0) return TB200_OK;   // nothing to read or write: empty tensors have no address
  if (!a->k || !a->v || !a->k_codes || !a->v_codes || !a->k_meta || !a->v_meta) return TB200_ERR_INVALID;
  if (!aligned16(a->k) || !aligned16(a->v) || !aligned16(a->k_codes) || !aligned16(a->v_codes) || !aligned16(a->k_meta) || !aligned16(a->v_meta))
    return TB200_ERR_INVALID;
  if (!aligned4(a->start) || !aligned4(a->n_rows)) return TB200_ERR_INVALID;
  const int64_t ext[3] = {a->batch, a->n_kv_heads, a->rows};
  if (check_strides(a->k_stride, ext, a->head_dim, false) != TB200_OK || check_strides(a->v_stride, ext, a->head_dim, false) != TB200_OK)
    return TB200_ERR_INVALID;
  return TB200_OK;
}

enum RowsWork { kAppend, kRead, kReadSeen };

RowsParams rows_params(const tb200_kv4_rows_args& a) {
  RowsParams p;
  memset(&p, 0, sizeof(p));
  p.start = a.start; p.n_rows = a.n_rows; p.start_all = a.start_all;
  p.rows = a.rows; p.heads = a.n_kv_heads; p.cache_len = a.cache_len;
  p.x[0] = static_cast<uint8_t*>(a.k);
  p.x[1] = static_cast<uint8_t*>(a.v);
  for (int i = 0; i < 3; ++i) { p.stride[0][i] = a.k_stride[i]; p.stride[1][i] = a.v_stride[i]; }
  p.codes[0] = static_cast<uint8_t*>(a.k_codes);
  p.codes[1] = static_cast<uint8_t*>(a.v_codes);
  p.meta[0] = static_cast<uint8_t*>(a.k_meta);
  p.meta[1] = static_cast<uint8_t*>(a.v_meta);
  return p;
}

template <typename T, int D>
int launch_rows(RowsParams p, int batch, RowsWork work, int num_sms, cudaStream_t stream) {
  p.n_bh = static_cast<long long>(batch) * p.heads;
  p.units = p.n_bh * ((p.rows + RowsShape<D>::kUnitRows - 1) / RowsShape<D>::kUnitRows);
  // several waves: the hardware deals CTAs out as SMs become free (8 per SM: 6 % slower)
  const long long most = static_cast<long long>(num_sms) * 32;
  const dim3 grid(static_cast<unsigned>(p.units < most ? p.units : most));
  cudaError_t e;
  if (work == kAppend) e = launch_chained(kv4_append_kernel<T, D>, grid, dim3(kThreads), 0, stream, p);
  else if (work == kRead) e = launch_chained(kv4_read_kernel<T, D, false>, grid, dim3(kThreads), 0, stream, p);
  else e = launch_chained(kv4_read_kernel<T, D, true>, grid, dim3(kThreads), 0, stream, p);
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? TB200_OK : TB200_ERR_CUDA;
}

int launch_rows(const RowsParams& p, int dtype, int head_dim, int batch, RowsWork work, int num_sms, cudaStream_t stream) {
  if (batch == 0 || p.rows == 0 || p.cache_len == 0) return TB200_OK;
  if (dtype == TB200_BF16)
    return head_dim == 128 ? launch_rows<__nv_bfloat16, 128>(p, batch, work, num_sms, stream) : launch_rows<__nv_bfloat16, 64>(p, batch, work, num_sms, stream);
  return head_dim == 128 ? launch_rows<__half, 128>(p, batch, work, num_sms, stream) : launch_rows<__half, 64>(p, batch, work, num_sms, stream);
}

}  // namespace

int launch_kv4_prompt_operands(const tb200_cache_attn_args& a, int window, int sinks, const Kv4PromptOperands& to, int num_sms, cudaStream_t stream) {
  RowsParams p;
  memset(&p, 0, sizeof(p));
  p.n_rows = a.kv_lens; p.rows = to.len; p.heads = a.n_kv_heads; p.cache_len = a.cache_len;
  p.n_bh = static_cast<long long>(a.batch) * a.n_kv_heads;
  p.x[0] = static_cast<uint8_t*>(to.k16);
  p.x[1] = static_cast<uint8_t*>(to.v16);
  for (int w = 0; w < 2; ++w) {
    p.stride[w][2] = a.head_dim;
    p.stride[w][1] = static_cast<long long>(to.len) * a.head_dim;
    p.stride[w][0] = p.stride[w][1] * a.n_kv_heads;
  }
  p.codes[0] = static_cast<uint8_t*>(const_cast<void*>(a.k_codes));
  p.codes[1] = static_cast<uint8_t*>(const_cast<void*>(a.v_codes));
  p.meta[0] = static_cast<uint8_t*>(const_cast<void*>(a.k_meta));
  p.meta[1] = static_cast<uint8_t*>(const_cast<void*>(a.v_meta));
  p.q_rows = a.q_rows; p.q_rows_max = a.rows; p.window = window; p.sinks = sinks; p.packed_head = to.packed_head;
  p.head_factor = reinterpret_cast<const float4*>(to.head_factor);
  if (a.dtype == TB200_BF16) {
    FactorParams f;
    f.rows = p;
    f.q = static_cast<const uint8_t*>(a.q);
    for (int i = 0; i < 3; ++i) f.q_stride[i] = a.q_stride[i];
    f.q16 = static_cast<uint8_t*>(to.q16);
    f.q_factor = to.q_factor;
    f.head_factor = reinterpret_cast<float4*>(to.head_factor);
    f.q_heads = a.n_q_heads;
    f.batch = a.batch;
    // a warp per row of q, at most sixteen CTAs' worth of them per SM over the whole batch
    const long long q_ctas = (static_cast<long long>(a.n_q_heads) * a.rows + kFactorThreads / 32 - 1) / (kFactorThreads / 32);
    const long long most = static_cast<long long>(num_sms) * 16 / a.batch + 1;
    const dim3 grid(static_cast<unsigned>(a.n_kv_heads + (q_ctas < most ? q_ctas : most)), static_cast<unsigned>(a.batch < 65535 ? a.batch : 65535));
    const cudaError_t e = a.head_dim == 128 ? launch_chained(kv4_factors_kernel<128>, grid, dim3(kFactorThreads), 0, stream, f)
                                            : launch_chained(kv4_factors_kernel<64>, grid, dim3(kFactorThreads), 0, stream, f);
    if (e != cudaSuccess || cudaGetLastError() != cudaSuccess) return TB200_ERR_CUDA;
  }
  return launch_rows(p, a.dtype, a.head_dim, a.batch, kReadSeen, num_sms, stream);
}

}  // namespace tb200

using namespace tb200;

extern "C" int tb200_kv4_rows_check(const tb200_kv4_rows_args* a) { return check_rows(a); }

extern "C" int tb200_kv4_append(const tb200_kv4_rows_args* a, void* stream) {
  const int bad = check_rows(a);
  if (bad != TB200_OK) return bad;
  const bool any = a->batch > 0 && a->rows > 0 && a->cache_len > 0;
  if (any && (a->k_codes == a->v_codes || a->k_meta == a->v_meta)) return TB200_ERR_INVALID;   // written from two sources
  int status = TB200_OK;
  DeviceState* st = device_state(&status);
  if (!st) return status;
  return launch_rows(rows_params(*a), a->dtype, a->head_dim, a->batch, kAppend, st->num_sms, static_cast<cudaStream_t>(stream));
}

extern "C" int tb200_kv4_read(const tb200_kv4_rows_args* a, void* stream) {
  const int bad = check_rows(a);
  if (bad != TB200_OK) return bad;
  const int64_t ext[3] = {a->batch, a->n_kv_heads, a->rows};   // k and v are written here
  const bool any = a->batch > 0 && a->rows > 0 && a->cache_len > 0;
  if (any && a->k == a->v) return TB200_ERR_INVALID;
  if (check_strides(a->k_stride, ext, a->head_dim, true) != TB200_OK || check_strides(a->v_stride, ext, a->head_dim, true) != TB200_OK)
    return TB200_ERR_INVALID;
  int status = TB200_OK;
  DeviceState* st = device_state(&status);
  if (!st) return status;
  return launch_rows(rows_params(*a), a->dtype, a->head_dim, a->batch, kRead, st->num_sms, static_cast<cudaStream_t>(stream));
}
