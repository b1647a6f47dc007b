// The 4-bit KV cache: rows are quantised as they are written (tb200_kv4_append) and turned back into 16-bit rows
// (tb200_kv4_read).  A group is 64 consecutive values x of a row; with lo = min x and s = (max x - min x) / 15 it is
// held as the codes c = round((x - lo) / s) and the pair (s, lo) in the cache's 16-bit type, and stands for lo + c s.
// 64 values take 32 + 4 bytes: 4.5 bits per value.
//
// Bound: HBM.  One row of D = 128 moves 256 + 72 bytes.  Eight lanes share a group (eight values, one 16-byte access
// each), so that minimum and maximum are three shuffles.
#include "common.cuh"
#include "internal.h"
#include "kv4.cuh"

namespace tb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 4;   // rows of a reading thread: eight loads in flight

struct RowsParams {
  const int32_t* start;
  const int32_t* n_rows;
  int start_all, rows, heads, cache_len, row_blocks;
  long long units;          // batch * heads * row_blocks
  uint8_t* x[2];            // k, v
  long long stride[2][3];   // elements: batch, head, row
  uint8_t* codes[2];
  uint8_t* meta[2];
  const int32_t* q_rows;    // SEEN
  int q_rows_max, window, sinks;
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

// Codes of eight values of a group (x - lo and s exact in 64 bits where a quotient lies next to a border).
template <typename T>
__device__ __forceinline__ uint32_t encode8(const uint4& raw, float lo, float s) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = Bits<T>::f((w[i >> 1] >> ((i & 1) * 16)) & 0xffffu);
    float c = 0.f;
    if (s > 0.f) c = static_cast<float>(fmin(fmax(rint((static_cast<double>(x) - static_cast<double>(lo)) / static_cast<double>(s)), 0.0), 15.0));
    word |= static_cast<uint32_t>(c) << (4 * i);
  }
  return word;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(const RowsParams p) {
  constexpr int kLanes = D / 8;                 // lanes per row
  constexpr int kRows = kThreads / kLanes;      // rows of a unit
  const int tid = threadIdx.x;
  const int r_in = tid / kLanes, c8 = tid % kLanes;
  for (long long u = blockIdx.x; u < p.units; u += gridDim.x) {
    const long long bh = u / p.row_blocks;
    const int rb = static_cast<int>(u - bh * p.row_blocks);
    const int b = static_cast<int>(bh / p.heads), h = static_cast<int>(bh - static_cast<long long>(b) * p.heads);
    const int row = rb * kRows + r_in;
    const int n = p.n_rows ? min(p.n_rows[b], p.rows) : p.rows;
    const long long pos = static_cast<long long>(p.start ? p.start[b] : p.start_all) + row;
    const bool live = row < n && pos >= 0 && pos < p.cache_len;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      uint4 raw = make_uint4(0u, 0u, 0u, 0u);
      if (live)
        raw = *reinterpret_cast<const uint4*>(p.x[which] + 2 * (b * p.stride[which][0] + h * p.stride[which][1] + row * p.stride[which][2] + c8 * 8));
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
      float lo = INFINITY, hi = -INFINITY;
      bool odd = false;   // an infinity or a NaN
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = Bits<T>::f((w[i >> 1] >> ((i & 1) * 16)) & 0xffffu);
        odd |= !(fabsf(x) < INFINITY);
        lo = fminf(lo, x);
        hi = fmaxf(hi, x);
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        odd |= __shfl_xor_sync(0xffffffffu, static_cast<int>(odd), o) != 0;
      }
      const float range = __fsub_rn(hi, lo);
      odd |= !(range < INFINITY);
      const uint32_t sb = odd ? 0x7fffu : Bits<T>::rn(__fdiv_rn(range, 15.f));
      const uint32_t lb = odd ? 0x7fffu : Bits<T>::rn(lo);
      if (live) {
        const long long crow = bh * p.cache_len + pos;
        const uint32_t word = encode8<T>(raw, lo, odd ? 0.f : Bits<T>::f(sb));
        *reinterpret_cast<uint32_t*>(p.codes[which] + crow * (D / 2) + c8 * 4) = word;
        if ((c8 & 7) == 0) *reinterpret_cast<uint32_t*>(p.meta[which] + (crow * (D / 64) + c8 / 8) * 4) = sb | (lb << 16);
      }
    }
  }
}

// SEEN: only the positions that some query row of the sequence sees (a prompt's attention reads the 16-bit rows next).
template <typename T, int D, bool SEEN>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const RowsParams p) {
  constexpr int kLanes = D / 8;
  constexpr int kRows = kThreads / kLanes;   // rows side by side
  if constexpr (SEEN) pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int r_in = tid / kLanes, c8 = tid % kLanes;
  for (long long u = blockIdx.x; u < p.units; u += gridDim.x) {
    const long long bh = u / p.row_blocks;
    const int rb = static_cast<int>(u - bh * p.row_blocks);
    const int b = static_cast<int>(bh / p.heads), h = static_cast<int>(bh - static_cast<long long>(b) * p.heads);
    const int n = p.n_rows ? min(p.n_rows[b], p.rows) : p.rows;
    const int start = p.start ? p.start[b] : p.start_all;
    int low = 0, few = 0;
    if constexpr (SEEN) {
      const int r = p.q_rows ? max(0, min(p.q_rows[b], p.q_rows_max)) : p.q_rows_max;
      low = p.window > 0 ? n - r - p.window + 1 : 0;
      few = r > 0 ? p.sinks : 0;
      if (r == 0) low = n;
    }
    uint32_t word[2][kPerThread], m[2][kPerThread];
    bool live[kPerThread];
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int row = (rb * kPerThread + k) * kRows + r_in;
      const long long pos = static_cast<long long>(start) + row;
      live[k] = row < n && pos >= 0 && pos < p.cache_len;
      if constexpr (SEEN) live[k] = live[k] && (row >= low || row < few);
      const long long crow = bh * p.cache_len + pos;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        word[w][k] = live[k] ? __ldg(reinterpret_cast<const uint32_t*>(p.codes[w] + crow * (D / 2) + c8 * 4)) : 0u;
        m[w][k] = live[k] ? __ldg(reinterpret_cast<const uint32_t*>(p.meta[w] + (crow * (D / 64) + c8 / 8) * 4)) : 0u;
      }
    }
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      if (!live[k]) continue;
      const long long row = (rb * kPerThread + k) * kRows + r_in;
#pragma unroll
      for (int w = 0; w < 2; ++w)
        *reinterpret_cast<uint4*>(p.x[w] + 2 * (b * p.stride[w][0] + h * p.stride[w][1] + row * p.stride[w][2] + c8 * 8)) =
            Kv4Decode<T>::decode8(word[w][k], m[w][k]);
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
  const int unit_rows = kThreads / (D / 8) * (work == kAppend ? 1 : kPerThread);
  p.row_blocks = (p.rows + unit_rows - 1) / unit_rows;
  p.units = static_cast<long long>(batch) * p.heads * p.row_blocks;
  const long long most = static_cast<long long>(num_sms) * 8;
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

int launch_kv4_read_seen(const tb200_cache_attn_args& a, int window, int sinks, void* k16, void* v16, int num_sms, cudaStream_t stream) {
  RowsParams p;
  memset(&p, 0, sizeof(p));
  p.n_rows = a.kv_lens; p.rows = a.cache_len; p.heads = a.n_kv_heads; p.cache_len = a.cache_len;
  p.x[0] = static_cast<uint8_t*>(k16);
  p.x[1] = static_cast<uint8_t*>(v16);
  for (int w = 0; w < 2; ++w) {
    p.stride[w][2] = a.head_dim;
    p.stride[w][1] = static_cast<long long>(a.cache_len) * a.head_dim;
    p.stride[w][0] = p.stride[w][1] * a.n_kv_heads;
  }
  p.codes[0] = static_cast<uint8_t*>(const_cast<void*>(a.k_codes));
  p.codes[1] = static_cast<uint8_t*>(const_cast<void*>(a.v_codes));
  p.meta[0] = static_cast<uint8_t*>(const_cast<void*>(a.k_meta));
  p.meta[1] = static_cast<uint8_t*>(const_cast<void*>(a.v_meta));
  p.q_rows = a.q_rows; p.q_rows_max = a.rows; p.window = window; p.sinks = sinks;
  return launch_rows(p, a.dtype, a.head_dim, a.batch, kReadSeen, num_sms, stream);
}

}  // namespace tb200

using namespace tb200;

extern "C" int tb200_kv4_rows_check(const tb200_kv4_rows_args* a) { return check_rows(a); }

extern "C" int tb200_kv4_append(const tb200_kv4_rows_args* a, void* stream) {
  const int bad = check_rows(a);
  if (bad != TB200_OK) return bad;
  int status = TB200_OK;
  DeviceState* st = device_state(&status);
  if (!st) return status;
  return launch_rows(rows_params(*a), a->dtype, a->head_dim, a->batch, kAppend, st->num_sms, static_cast<cudaStream_t>(stream));
}

extern "C" int tb200_kv4_read(const tb200_kv4_rows_args* a, void* stream) {
  const int bad = check_rows(a);
  if (bad != TB200_OK) return bad;
  const int64_t ext[3] = {a->batch, a->n_kv_heads, a->rows};   // k and v are written here
  if (check_strides(a->k_stride, ext, a->head_dim, true) != TB200_OK || check_strides(a->v_stride, ext, a->head_dim, true) != TB200_OK)
    return TB200_ERR_INVALID;
  int status = TB200_OK;
  DeviceState* st = device_state(&status);
  if (!st) return status;
  return launch_rows(rows_params(*a), a->dtype, a->head_dim, a->batch, kRead, st->num_sms, static_cast<cudaStream_t>(stream));
}
