// What the decode kernels over caches (attn_cache.cu: 4 bits, attn_win.cu: 16 bits) share: the line of key tiles and how it
// is dealt out over the CTAs, and the merging of partial results.
//
//   unit     (sequence, kv head, R query rows): the rows of a unit are (new token, query head of the group) pairs, so
//            that a cache row is read once for all query heads that share it.
//   line     the key tiles of all units, one after the other, dealt out in equal stretches over the CTAs (each computes
//            the line's layout from kv_lens itself): long and short sequences load the SMs evenly, with no host knowledge
//            of the lengths.  A unit that lies within one CTA's stretch is finished there; the others leave a partial
//            result (accumulator, maximum, sum) per stretch, which cache_combine_kernel merges in the order of the keys.
//   warp     takes every fourth tile of a stretch.
//   cluster  with few keys a unit is one cluster's instead: C CTAs (1, 2, 4 or 8) share its tiles evenly and merge their
//            results through distributed shared memory.  One launch, no scratch: one token on 1037 positions, 32/8 heads,
//            takes 7.0 us of device time instead of 13.3.
#pragma once

#include <math.h>

#include "common.cuh"
#include "internal.h"

namespace tb200 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;   // the exponent reference of a row moves only when its maximum has grown by more than 2^kSlack
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

struct CacheAttnParams {
  int B, S, Hq, Hkv, group, cache_len, window, sinks;
  int row_tiles;             // units per (sequence, kv head) at most
  int cluster;               // 0: the line; else CTAs per unit
  int record_per_unit;       // the line: what `split` is indexed by, the unit where there are no more units than stretches,
                             // else the stretch
  float scale_log2;
  const uint8_t* q;
  uint8_t* o;
  long long qs[3], os[3];
  const int32_t* kv_lens;
  const int32_t* q_rows;
  const uint8_t *k_codes, *v_codes, *k_meta, *v_meta;
  float* part_o;             // (2 grid, R, D)
  float* part_ml;            // (2 grid, R, 2)
  int4* split;               // (grid) units that lie in several stretches and in how many (0: no such unit): by stretch
                             // (sequence, kv head, row tile, how many), for the one that begins there and goes on; by unit
                             // (stretch it begins in, -, -, how many)
  int stretches;             // CTAs of the decode kernel
  int* err;
  long long wait_limit;
};

// What a sequence asks for.
struct Seq {
  int n, r;                  // positions, new rows
  int few;                   // first positions that stay visible, below the window
  int sink_tiles, win_tile;  // tiles [0, sink_tiles) and from win_tile on
  int tiles;                 // tiles of a unit
  int units;                 // units of the sequence: kv heads x row tiles
};
__device__ __forceinline__ Seq load_seq(const CacheAttnParams& p, int b, int tile, int unit_rows) {
  Seq s;
  s.n = max(0, min(__ldg(p.kv_lens + b), p.cache_len));
  s.r = p.q_rows ? max(0, min(__ldg(p.q_rows + b), p.S)) : p.S;
  const int low = p.window > 0 ? max(0, s.n - s.r - p.window + 1) : 0;
  s.few = min(p.sinks, low);
  s.win_tile = low / tile;
  s.sink_tiles = min((s.few + tile - 1) / tile, s.win_tile);
  s.tiles = max(1, s.sink_tiles + (s.n + tile - 1) / tile - s.win_tile);   // a sequence without keys: one masked tile writes the zeros
  s.units = s.r > 0 ? p.Hkv * ((s.r * p.group + unit_rows - 1) / unit_rows) : 0;
  return s;
}

// The line of all tiles: its length, and how it is dealt out.  Every lane of a warp calls these and gets the same.
struct Line {
  int total;    // tiles of all units
  int per;      // tiles of a stretch
  int seq;      // the sequence in which position x lies
  int base;     // the line's position of that sequence's first tile
};
// x is the first position of stretch `stretch` (behind the line's end: seq and base are not set).
__device__ __forceinline__ Line walk_line(const CacheAttnParams& p, int tile, int unit_rows, int min_tiles, int stretch) {
  const int lane = static_cast<int>(lane_id());
  Line ln;
  ln.seq = ln.base = 0;
  int sum = 0, own = 0, total = 0;
  auto scan = [&](int b0) {   // inclusive sums over 32 sequences
    const int b = b0 + lane;
    own = 0;
    if (b < p.B) {
      const Seq s = load_seq(p, b, tile, unit_rows);
      own = s.tiles * s.units;
    }
    sum = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += up;
    }
  };
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    scan(b0);
    total += __shfl_sync(0xffffffffu, sum, 31);
  }
  ln.total = total;
  ln.per = max((total + p.stretches - 1) / p.stretches, min_tiles);
  const int x = ln.per * stretch;
  if (x >= total) return ln;
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    if (p.B > 32) scan(b0);   // else the sums are still there
    const unsigned hit = __ballot_sync(0xffffffffu, before + sum > x);
    if (hit) {
      const int l = __ffs(hit) - 1;
      ln.seq = b0 + l;
      ln.base = before + __shfl_sync(0xffffffffu, sum - own, l);
      break;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return ln;
}

// One segment: the part of a unit that lies in this CTA's stretch.
struct Segment {
  int b, h, rt;              // sequence, kv head, row tile
  int v0, v1;                // tiles of the unit
  int n_rows;                // query rows of the (sequence, kv head)
};
// The CTA's walk along its stretch.
struct Walk {
  Line ln;
  Seq sq;
  int x, x_end;              // positions on the line: of the current segment, of the stretch's end
  int base, b;               // the line's position of the sequence's first tile; the sequence
  Segment own;               // cluster: this CTA's share of its unit
  __device__ __forceinline__ bool begin(const CacheAttnParams& p, int tile, int unit_rows, int min_tiles) {   // false: nothing to do
    if (p.cluster > 0) {
      int u = static_cast<int>(blockIdx.x) / p.cluster;
      const int rank = static_cast<int>(blockIdx.x) - u * p.cluster;
      own.rt = u % p.row_tiles;
      u /= p.row_tiles;
      own.h = u % p.Hkv;
      own.b = u / p.Hkv;
      sq = load_seq(p, own.b, tile, unit_rows);
      own.n_rows = sq.r * p.group;
      if (own.rt * unit_rows >= own.n_rows) return false;   // every CTA of the cluster
      const int per = (sq.tiles + p.cluster - 1) / p.cluster;
      own.v0 = min(sq.tiles, rank * per);
      own.v1 = min(sq.tiles, own.v0 + per);
      x = 0;
      x_end = 1;
      return true;
    }
    ln = walk_line(p, tile, unit_rows, min_tiles, blockIdx.x);
    x = ln.per * static_cast<int>(blockIdx.x);
    x_end = min(x + ln.per, ln.total);
    if (x >= x_end) {
      if (threadIdx.x == 0 && !p.record_per_unit) p.split[blockIdx.x] = make_int4(0, 0, 0, 0);
      return false;
    }
    base = ln.base;
    b = ln.seq;
    sq = load_seq(p, b, tile, unit_rows);
    return true;
  }
  __device__ __forceinline__ void advance(const CacheAttnParams& p, const Segment& s) { x += p.cluster > 0 ? 1 : s.v1 - s.v0; }
  __device__ __forceinline__ Segment segment(const CacheAttnParams& p, int tile, int unit_rows) {
    if (p.cluster > 0) return own;
    while (x >= base + sq.tiles * sq.units) {
      base += sq.tiles * sq.units;
      sq = load_seq(p, ++b, tile, unit_rows);
    }
    Segment s;
    const int unit = (x - base) / sq.tiles;
    s.v0 = x - base - unit * sq.tiles;
    s.v1 = min(sq.tiles, s.v0 + x_end - x);
    const int rts = sq.units / p.Hkv;
    s.b = b;
    s.h = unit / rts;
    s.rt = unit - s.h * rts;
    s.n_rows = sq.r * p.group;
    return s;
  }
  __device__ __forceinline__ int tile_of(int v) const { return v < sq.sink_tiles ? v : sq.win_tile + v - sq.sink_tiles; }
};

// Shared memory in which the warps leave their shares of a segment.
template <int D, int NT> struct MergeSmem {
  static constexpr int kR = 8 * NT;
  static constexpr int kPitch = D + 4;                       // floats per row: 4 keep the rows' banks apart
  static constexpr int kMlOff = kWarps * kR * kPitch * 4;    // float2 [warps][R] behind float [warps][R][pitch]
  static constexpr int kBytes = kMlOff + kWarps * kR * 8;
};
// A CTA's share of a unit, for its cluster.
template <int D, int R> struct ShareSmem {
  static constexpr int kMlOff = R * D * 4;                   // float2 [R] behind float [R][D]
  static constexpr int kBytes = kMlOff + R * 8;
};
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_f32x2(uint32_t cluster_addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_addr) : "memory");
  return v;
}
// Columns d to d + 3 of the unit's row m, divided by its sum, into o.
template <typename T, int R>
__device__ __forceinline__ void store_row(const CacheAttnParams& p, const Segment& sg, int m, int d, const float4& acc, float sum) {
  const int mr = sg.rt * R + m;
  if (mr >= sg.n_rows) return;
  const float inv = sum > 0.f ? 1.f / sum : sum;   // 0: the row sees nothing; NaN stays
  const int tok = mr / p.group;
  T* op = reinterpret_cast<T*>(p.o) + sg.b * p.os[0] + (sg.h * p.group + mr - tok * p.group) * p.os[1] + tok * p.os[2] + d;
  *reinterpret_cast<uint2*>(op) = make_uint2(Pack2<T>::pack(acc.x * inv, acc.y * inv), Pack2<T>::pack(acc.z * inv, acc.w * inv));
}

// The four warps' shares (of each row H from each warp) in a fixed order: into o where the unit lies in this stretch
// altogether, else into the stretch's partial results, or with a cluster into `share` and from there, all CTAs' in the order
// of their keys, into o.  Called by the whole CTA, with the shares written and a barrier behind them.
template <typename T, int D, int NT, int H>
__device__ __forceinline__ void merge_segment(const CacheAttnParams& p, const uint8_t* smem, uint8_t* share, const Walk& wk, const Segment& sg) {
  using M = MergeSmem<D, NT>;
  constexpr int R = M::kR / H;
  using S = ShareSmem<D, R>;
  const bool whole = p.cluster > 0 ? p.cluster == 1 : sg.v0 == 0 && sg.v1 == wk.sq.tiles;
  if (p.cluster == 0 && threadIdx.x == 0) {
    const int c = static_cast<int>(blockIdx.x), parts = sg.v0 == 0 && !whole ? (wk.x + wk.sq.tiles - 1) / wk.ln.per - c + 1 : 0;
    if (p.record_per_unit) {
      if (sg.v0 == 0) p.split[(sg.b * p.Hkv + sg.h) * p.row_tiles + sg.rt] = make_int4(c, 0, 0, parts);
    } else if (wk.x + sg.v1 - sg.v0 >= wk.x_end) {   // the stretch's last segment
      p.split[c] = make_int4(sg.b, sg.h, sg.rt, parts);
    }
  }
  const float* mall = reinterpret_cast<const float*>(smem);
  const float2* mlall = reinterpret_cast<const float2*>(smem + M::kMlOff);
  const int slot_out = 2 * blockIdx.x + (sg.v0 == 0 ? 1 : 0);
  for (int i = threadIdx.x; i < R * D / 4; i += kThreads) {
    const int m = i / (D / 4), d = (i % (D / 4)) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps * H; ++w) top = fmaxf(top, mlall[w * R + m].x);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps * H; ++w) {
      const float2 ml = mlall[w * R + m];
      const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
      const float4 a = *reinterpret_cast<const float4*>(mall + (w * R + m) * M::kPitch + d);
      sum = fmaf(f, ml.y, sum);
      acc.x = fmaf(f, a.x, acc.x); acc.y = fmaf(f, a.y, acc.y); acc.z = fmaf(f, a.z, acc.z); acc.w = fmaf(f, a.w, acc.w);
    }
    if (whole) {
      store_row<T, R>(p, sg, m, d, acc, sum);
    } else if (p.cluster > 0) {
      *reinterpret_cast<float4*>(share + i * 16) = acc;
      if (d == 0) *reinterpret_cast<float2*>(share + S::kMlOff + m * 8) = make_float2(top, sum);
    } else {
      *reinterpret_cast<float4*>(p.part_o + (static_cast<long long>(slot_out) * R + m) * D + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (static_cast<long long>(slot_out) * R + m) * 2) = make_float2(top, sum);
    }
  }
  if (p.cluster <= 1) return;
  cluster_sync_all();
  const int rank = static_cast<int>(cluster_ctarank());
  const uint32_t base = smem_u32(share);
  for (int i = rank * kThreads + threadIdx.x; i < R * D / 4; i += p.cluster * kThreads) {
    const int m = i / (D / 4), d = (i % (D / 4)) * 4;
    float2 ml[8];
    float4 a[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {   // all loads under way at once
      ml[r] = make_float2(-INFINITY, 0.f);
      a[r] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < p.cluster) {
        const uint32_t peer = mapa_u32(base, r);
        ml[r] = ld_cluster_f32x2(peer + S::kMlOff + m * 8);
        a[r] = ld_cluster_f32x4(peer + i * 16);
      }
    }
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) top = fmaxf(top, ml[r].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float f = ml[r].x == -INFINITY ? 0.f : fast_exp2(ml[r].x - top);
      sum = fmaf(f, ml[r].y, sum);
      acc.x = fmaf(f, a[r].x, acc.x); acc.y = fmaf(f, a[r].y, acc.y); acc.z = fmaf(f, a[r].z, acc.z); acc.w = fmaf(f, a[r].w, acc.w);
    }
    store_row<T, R>(p, sg, m, d, acc, sum);
  }
  cluster_sync_all();   // nobody's shared memory goes away while a peer still reads it
}

// The launch of a decode kernel: p.stretches CTAs, in clusters where the parameters say so.
template <typename... KArgs, typename... Args>
inline int launch_decode_grid(void (*kernel)(KArgs...), const CacheAttnParams& p, size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(p.stretches));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (p.cluster > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(p.cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if (chain_next_launch()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args&&>(args)...) == cudaSuccess && cudaGetLastError() == cudaSuccess ? TB200_OK : TB200_ERR_CUDA;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// attn_cache.cu
int launch_cache_combine(const CacheAttnParams& p, int dtype, int head_dim, int unit_rows, cudaStream_t stream);
// attn_win.cu: the decode kernel over 16-bit caches, in a ChainScope; p.stretches as cache16_stretches says
int launch_cache16(const CacheAttnParams& p, const tb200_cache_attn_args& a, int unit_rows, cudaStream_t stream);   // 8 or 16
int cache16_stretches(int num_sms);

}  // namespace tb200
