// Attention over a cache that already holds the new rows: tb200_attn_window (16-bit caches) and tb200_kv4_attn (4-bit
// caches), per-sequence lengths, an optional sliding window with a few first positions that stay visible.
//
// One warp per (sequence, query head, query row): the keys one after the other, running maximum and sum.
#include <math.h>

#include "common.cuh"
#include "internal.h"
#include "kv4.cuh"

namespace tb200 {

namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct CacheAttnParams {
  int B, S, Hq, Hkv, cache_len, window, sinks;
  float scale_log2;
  const uint8_t* q;
  uint8_t* o;
  long long qs[3], os[3];
  const int32_t* kv_lens;
  const int32_t* q_rows;
  const uint8_t* k16;
  const uint8_t* v16;
  long long ks[3], vs[3];
  const uint8_t *k_codes, *v_codes, *k_meta, *v_meta;
};

template <typename T> __device__ __forceinline__ float to_f(T x) { return static_cast<float>(x); }

template <typename T, int D, bool KV4>
__global__ void __launch_bounds__(kThreads) cache_attn_kernel(const CacheAttnParams p) {
  constexpr int V = D / 32;   // columns per lane
  const int lane = threadIdx.x & 31;
  const long long rows = static_cast<long long>(p.B) * p.Hq * p.S;
  const long long step = static_cast<long long>(gridDim.x) * (kThreads / 32);
  for (long long w = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); w < rows; w += step) {
    const int i = static_cast<int>(w % p.S);
    const int hq = static_cast<int>((w / p.S) % p.Hq);
    const int b = static_cast<int>(w / (static_cast<long long>(p.S) * p.Hq));
    const int n = max(0, min(p.kv_lens[b], p.cache_len));
    const int r = p.q_rows ? max(0, min(p.q_rows[b], p.S)) : p.S;
    if (i >= r) continue;
    const int hkv = hq / (p.Hq / p.Hkv);
    const int at = n - r + i;
    const int low = p.window > 0 ? max(0, at - p.window + 1) : 0;
    const int few = min(p.sinks, low);
    float q[V], o[V];
    const T* qp = reinterpret_cast<const T*>(p.q) + b * p.qs[0] + hq * p.qs[1] + i * p.qs[2] + lane * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      q[e] = to_f(qp[e]) * p.scale_log2;
      o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int x = 0; x < few + at + 1 - low; ++x) {
      const int j = x < few ? x : x - few + low;
      float k[V], v[V];
      if constexpr (KV4) {
        const long long row = (static_cast<long long>(b) * p.Hkv + hkv) * p.cache_len + j;
        const int c0 = lane * V;
        const T* km = reinterpret_cast<const T*>(p.k_meta) + (row * (D / 64) + c0 / 64) * 2;
        const T* vm = reinterpret_cast<const T*>(p.v_meta) + (row * (D / 64) + c0 / 64) * 2;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int sh = ((c0 + e) & 1) * 4;
          k[e] = fmaf(static_cast<float>((p.k_codes[row * (D / 2) + (c0 + e) / 2] >> sh) & 15), to_f(km[0]), to_f(km[1]));
          v[e] = fmaf(static_cast<float>((p.v_codes[row * (D / 2) + (c0 + e) / 2] >> sh) & 15), to_f(vm[0]), to_f(vm[1]));
        }
      } else {
        const T* kp = reinterpret_cast<const T*>(p.k16) + b * p.ks[0] + hkv * p.ks[1] + j * p.ks[2] + lane * V;
        const T* vp = reinterpret_cast<const T*>(p.v16) + b * p.vs[0] + hkv * p.vs[1] + j * p.vs[2] + lane * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          k[e] = to_f(kp[e]);
          v[e] = to_f(vp[e]);
        }
      }
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) s = fmaf(q[e], k[e], s);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      const float m_new = fmaxf(m, s);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float a = fast_exp2(m - m_use), pr = fast_exp2(s - m_use);
      m = m_new;
      l = fmaf(l, a, pr);
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = fmaf(o[e], a, pr * v[e]);
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    T* op = reinterpret_cast<T*>(p.o) + b * p.os[0] + hq * p.os[1] + i * p.os[2] + lane * V;
#pragma unroll
    for (int e = 0; e < V; e += 2) *reinterpret_cast<uint32_t*>(op + e) = Pack2<T>::pack(o[e] * inv, o[e + 1] * inv);
  }
}

int check_attn(const tb200_cache_attn_args* a, bool kv4) {
  if (a == nullptr) return TB200_ERR_INVALID;
  if (a->dtype != TB200_BF16 && a->dtype != TB200_F16) return TB200_ERR_UNSUPPORTED;
  if (a->head_dim != 64 && a->head_dim != 128) return TB200_ERR_UNSUPPORTED;
  if (a->batch < 0 || a->rows < 0 || a->n_kv_heads < 1 || a->n_q_heads < 1 || a->n_q_heads % a->n_kv_heads || a->cache_len < 1) return TB200_ERR_INVALID;
  if (a->window < 0 || a->sinks < 0 || !(a->sm_scale > 0.f) || !(a->sm_scale < INFINITY)) return TB200_ERR_INVALID;
  if (!a->q || !a->o || !a->kv_lens || a->q == a->o || !aligned16(a->q) || !aligned16(a->o) || !aligned4(a->kv_lens) || !aligned4(a->q_rows))
    return TB200_ERR_INVALID;
  const int64_t ext[3] = {a->batch, a->n_q_heads, a->rows};
  if (check_strides(a->q_stride, ext, a->head_dim, false) != TB200_OK || check_strides(a->o_stride, ext, a->head_dim, true) != TB200_OK)
    return TB200_ERR_INVALID;
  if (kv4) {
    if ((a->cache_len & 3) || !a->k_codes || !a->v_codes || !a->k_meta || !a->v_meta) return TB200_ERR_INVALID;
    if (!aligned16(a->k_codes) || !aligned16(a->v_codes) || !aligned16(a->k_meta) || !aligned16(a->v_meta)) return TB200_ERR_INVALID;
  } else {
    if (!a->k_cache || !a->v_cache || !aligned16(a->k_cache) || !aligned16(a->v_cache)) return TB200_ERR_INVALID;
    const int64_t cext[3] = {a->batch, a->n_kv_heads, a->cache_len};
    if (check_strides(a->k_stride, cext, a->head_dim, false) != TB200_OK || check_strides(a->v_stride, cext, a->head_dim, false) != TB200_OK)
      return TB200_ERR_INVALID;
  }
  return TB200_OK;
}

template <typename T, int D, bool KV4>
int launch_simple(const CacheAttnParams& p, int num_sms, cudaStream_t stream) {
  const long long rows = static_cast<long long>(p.B) * p.Hq * p.S;
  long long blocks = (rows + kThreads / 32 - 1) / (kThreads / 32);
  if (blocks > num_sms * 8) blocks = num_sms * 8;
  cache_attn_kernel<T, D, KV4><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? TB200_OK : TB200_ERR_CUDA;
}

int run_attn(const tb200_cache_attn_args* a, bool kv4, void* stream_) {
  const int bad = check_attn(a, kv4);
  if (bad != TB200_OK) return bad;
  int status = TB200_OK;
  DeviceState* st = device_state(&status);
  if (!st) return status;
  if (a->batch == 0 || a->rows == 0) return TB200_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  CacheAttnParams p;
  p.B = a->batch; p.S = a->rows; p.Hq = a->n_q_heads; p.Hkv = a->n_kv_heads; p.cache_len = a->cache_len;
  p.window = a->window; p.sinks = a->window > 0 ? a->sinks : 0;
  p.scale_log2 = a->sm_scale * kLog2e;
  p.q = static_cast<const uint8_t*>(a->q);
  p.o = static_cast<uint8_t*>(a->o);
  for (int i = 0; i < 3; ++i) { p.qs[i] = a->q_stride[i]; p.os[i] = a->o_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; }
  p.kv_lens = a->kv_lens; p.q_rows = a->q_rows;
  p.k16 = static_cast<const uint8_t*>(a->k_cache);
  p.v16 = static_cast<const uint8_t*>(a->v_cache);
  p.k_codes = static_cast<const uint8_t*>(a->k_codes);
  p.v_codes = static_cast<const uint8_t*>(a->v_codes);
  p.k_meta = static_cast<const uint8_t*>(a->k_meta);
  p.v_meta = static_cast<const uint8_t*>(a->v_meta);
  const bool d128 = a->head_dim == 128;
  if (a->dtype == TB200_BF16) {
    if (kv4) return d128 ? launch_simple<__nv_bfloat16, 128, true>(p, st->num_sms, stream) : launch_simple<__nv_bfloat16, 64, true>(p, st->num_sms, stream);
    return d128 ? launch_simple<__nv_bfloat16, 128, false>(p, st->num_sms, stream) : launch_simple<__nv_bfloat16, 64, false>(p, st->num_sms, stream);
  }
  if (kv4) return d128 ? launch_simple<__half, 128, true>(p, st->num_sms, stream) : launch_simple<__half, 64, true>(p, st->num_sms, stream);
  return d128 ? launch_simple<__half, 128, false>(p, st->num_sms, stream) : launch_simple<__half, 64, false>(p, st->num_sms, stream);
}

}  // namespace
}  // namespace tb200

using namespace tb200;

extern "C" {

int tb200_attn_window_check(const tb200_cache_attn_args* a) { return check_attn(a, false); }
int tb200_kv4_attn_check(const tb200_cache_attn_args* a) { return check_attn(a, true); }
size_t tb200_attn_window_workspace_bytes(const tb200_cache_attn_args*) { return 0; }
size_t tb200_kv4_attn_workspace_bytes(const tb200_cache_attn_args*) { return 0; }
int tb200_attn_window(const tb200_cache_attn_args* a, void* stream) { return run_attn(a, false, stream); }
int tb200_kv4_attn(const tb200_cache_attn_args* a, void* stream) { return run_attn(a, true, stream); }

}  // extern "C"
