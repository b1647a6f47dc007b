// Attention of few query rows per sequence over 16-bit caches with per-sequence lengths and an optional sliding window:
// the decode form of tb200_attn_window (units, line and stretches: cache_line.cuh).
//
// Bound: HBM, the visible cache rows are read once per key/value head; a window makes calls short, so launch latency next.
// One token of 32 sequences of 1 to 4096 positions, window 1024 and 4 first ones, 32/8 heads of 128, bf16: 24.7 us for 133 MB,
// 82 % of the copy bandwidth.
// Sixteen keys per tile and warp: K and V arrive as TMA boxes of 16 keys x 64 columns (128-byte swizzle) in the warp's own
// ring, S^T = K Q^T and O^T = V^T P^T are m16n8k16 MMAs with the query rows as the 8 columns (a 16-row tile of queries
// would be half empty at eight query heads per key/value head), P goes from one to the other through movmatrix.
// Probabilities are rounded to the cache's type for the second product; their sum is taken before that, in fp32.
#include "cache_line.cuh"

namespace tb200 {

namespace {

constexpr int kTile = 16;
constexpr int kMinTiles = 2 * kWarps;

struct CacheMaps {
  CUtensorMap k, v;   // (B, Hkv, cache_len, D), boxes of 16 keys x 64 columns
};

template <int D, int NT> struct Smem16 {
  static constexpr int kBox = kTile * 128;                 // bytes
  static constexpr int kHalf = D / 64 * kBox;              // K or V of a tile
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kBarOff = kWarps * kStages * kStage;
  static_assert(MergeSmem<D, NT>::kBytes <= kBarOff, "the merge buffers must fit where the rings were");
  static constexpr int kShareOff = kBarOff + kWarps * kStages * 8 + 16;
  static constexpr int kTotal = kShareOff + ShareSmem<D, 8 * NT>::kBytes + 1024;   // + slack to align the base to 1 KiB
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (IsBf16<T>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, 2) cache_decode16_kernel(const __grid_constant__ CacheAttnParams p, const __grid_constant__ CacheMaps maps) {
  using L = Smem16<D, NT>;
  constexpr int R = 8 * NT, kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (kStages * L::kStage);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff) + warp * kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kBarOff + kWarps * kStages * 8);
  const AbortCtx ctx{p.err, abort_flag, p.wait_limit};
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[i], 1);
    if (warp == 0) {
      *abort_flag = 0;
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.v);
    }
    fence_mbar_init();
  }
  __syncthreads();

  Walk wk;
  if (!wk.begin(p, kTile, R, kMinTiles)) return;
  uint32_t used = 0;    // tiles this warp has taken through its ring
  bool ok = true;

  while (wk.x < wk.x_end) {
    const Segment sg = wk.segment(p, kTile, R);
    const Seq& sq = wk.sq;
    auto issue = [&](int v, uint32_t slot) {   // whole warp: one box per lane
      if (lane == 0) mbar_arrive_expect_tx(&bars[slot], L::kStage);
      __syncwarp();
      if (lane < 2 * (D / 64)) {
        const int dc = lane % (D / 64);
        tma_load_4d(ring + slot * L::kStage + lane * L::kBox, lane < D / 64 ? &maps.k : &maps.v, &bars[slot], dc * 64, wk.tile_of(v) * kTile, sg.h, sg.b);
      }
    };
    auto drain = [&](int v) {   // a wait gave up: the copies in flight (tile v and those behind it) get their time to land
      for (int i = 0; i < kStages && v + i * kWarps < sg.v1; ++i) {
        const uint32_t u = used + i;
        const long long t0 = clock64();
        while (!mbar_try_wait(&bars[u % kStages], (u / kStages) & 1) && clock64() - t0 < p.wait_limit) {
        }
      }
    };
    if (ok) {
#pragma unroll
      for (int i = 0; i < kStages; ++i)
        if (sg.v0 + warp + i * kWarps < sg.v1) issue(sg.v0 + warp + i * kWarps, (used + i) % kStages);
    }

    // ---- the unit's query rows: MMA column m is row rt * R + m, i.e. (token, query head of the group)
    uint32_t qf[NT][D / 16][2];
    int cpos[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int m = sg.rt * R + nt * 8 + g;
      const bool live = m < sg.n_rows;
      const int tok = live ? m / p.group : 0;
      const int hq = sg.h * p.group + (live ? m - tok * p.group : 0);
      const T* qp = reinterpret_cast<const T*>(p.q) + sg.b * p.qs[0] + hq * p.qs[1] + tok * p.qs[2] + 2 * t;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[nt][ks][0] = live ? __ldg(reinterpret_cast<const uint32_t*>(qp + ks * 16)) : 0u;
        qf[nt][ks][1] = live ? __ldg(reinterpret_cast<const uint32_t*>(qp + ks * 16 + 8)) : 0u;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int mc = sg.rt * R + nt * 8 + 2 * t + c;
        cpos[nt][c] = mc < sg.n_rows ? sq.n - sq.r + mc / p.group : -1;
      }
    }
    float o[NT][D / 16][4], l[NT][2], mx[NT][2], shift[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l[nt][c] = shift[nt][c] = 0.f;
        mx[nt][c] = -INFINITY;
      }
    }
    const int mat = lane >> 3, mrow = lane & 7;

    for (int v = sg.v0 + warp; v < sg.v1; v += kWarps) {
      const uint32_t slot = used % kStages;
      if (!ok || !mbar_wait(&bars[slot], (used / kStages) & 1, ctx, 711)) {   // (the CTA goes on to its barriers without this warp's keys)
        if (ok) drain(v);
        ok = false;
        break;
      }
      const uint32_t kbase = smem_u32(ring + slot * L::kStage), vbase = kbase + L::kHalf;
      const int k0 = wk.tile_of(v) * kTile;
      // every key of the tile visible to every row of the sequence?
      const bool full = k0 + kTile - 1 <= sq.n - sq.r && (p.window == 0 || k0 > sq.n - 1 - p.window || k0 + kTile - 1 < p.sinks);

      float s[NT][4];   // keys g (rows 2t, 2t + 1) and g + 8
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
      {
        const int key = (mat & 1) * 8 + mrow;
        const uint32_t row = kbase + key * 128;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const int piece = 2 * ks + (mat >> 1);   // 16-byte piece of the key's row; piece j of a 128-byte row r sits at j ^ (r & 7)
          uint32_t a[4];
          ldmatrix_x4(a, row + (piece >> 3) * L::kBox + (((piece & 7) ^ (key & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma<T>(s[nt], a, qf[nt][ks][0], qf[nt][ks][1]);
        }
      }
      uint32_t keep01 = 0xffffffffu, keep23 = 0xffffffffu;   // V of keys 2t, 2t + 1 and 2t + 8, 2t + 9
      if (!full) {
        auto sees = [&](int key, int pos) { return key <= pos && (p.window == 0 || key > pos - p.window || key < p.sinks); };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (!sees(k0 + g, cpos[nt][c])) s[nt][c] = -INFINITY;
            if (!sees(k0 + g + 8, cpos[nt][c])) s[nt][2 + c] = -INFINITY;
          }
        // a row of V that nobody sees may hold anything: 0 * inf and 0 * NaN must not arise
        auto alive = [&](int key) { return key < sq.n && (p.window == 0 || key > sq.n - sq.r - p.window || key < p.sinks); };
        keep01 = (alive(k0 + 2 * t) ? 0xffffu : 0u) | (alive(k0 + 2 * t + 1) ? 0xffff0000u : 0u);
        keep23 = (alive(k0 + 2 * t + 8) ? 0xffffu : 0u) | (alive(k0 + 2 * t + 9) ? 0xffff0000u : 0u);
      }
      // ---- running maximum: what a thread sees of it decides whether the warp has to look closer
      float top[NT][2];
      bool grown = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          top[nt][c] = fmaxf(s[nt][c], s[nt][2 + c]) * p.scale_log2;
          grown |= top[nt][c] > mx[nt][c] + kSlack;
        }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float m_new = top[nt][c];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, d));
            m_new = fmaxf(m_new, mx[nt][c]);
            const float a = m_new == -INFINITY ? 1.f : fast_exp2(mx[nt][c] - m_new);
            mx[nt][c] = m_new;
            shift[nt][c] = m_new == -INFINITY ? 0.f : -m_new;
            l[nt][c] *= a;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              o[nt][i][c] *= a;
              o[nt][i][2 + c] *= a;
            }
          }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          s[nt][c] = fast_exp2(fmaf(s[nt][c], p.scale_log2, shift[nt][c]));
          s[nt][2 + c] = fast_exp2(fmaf(s[nt][2 + c], p.scale_log2, shift[nt][c]));
          l[nt][c] += s[nt][c] + s[nt][2 + c];
        }
        pf[nt][0] = transpose8x8(Pack2<T>::pack(s[nt][0], s[nt][1]));
        pf[nt][1] = transpose8x8(Pack2<T>::pack(s[nt][2], s[nt][3]));
      }
      {
        const int key = (mat >> 1) * 8 + mrow;
        const uint32_t row = vbase + key * 128;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int piece = 2 * i + (mat & 1);
          uint32_t a[4];
          ldmatrix_x4_trans(a, row + (piece >> 3) * L::kBox + (((piece & 7) ^ (key & 7)) << 4));
          if (!full) {
            a[0] &= keep01; a[1] &= keep01;
            a[2] &= keep23; a[3] &= keep23;
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma<T>(o[nt][i], a, pf[nt][0], pf[nt][1]);
        }
      }
      __syncwarp();   // every lane has read the slot
      if (v + kStages * kWarps < sg.v1) issue(v + kStages * kWarps, slot);
      ++used;
    }

    // ---- this warp's share of the segment into shared memory: o relative to its own maximum
    __syncthreads();   // every warp is done with its ring
    using M = MergeSmem<D, NT>;
    float* wm = reinterpret_cast<float*>(smem) + warp * R * M::kPitch;
    float2* wml = reinterpret_cast<float2*>(smem + M::kMlOff) + warp * R;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int m = nt * 8 + 2 * t + c;
        float ls = l[nt][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, d);
        if (g == 0) wml[m] = make_float2(mx[nt][c], ls);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          wm[m * M::kPitch + i * 16 + g] = o[nt][i][c];
          wm[m * M::kPitch + i * 16 + g + 8] = o[nt][i][2 + c];
        }
      }
    __syncthreads();
    merge_segment<T, D, NT, 1>(p, smem, smem + L::kShareOff, wk, sg);
    fence_proxy_async_smem();   // the next copies overwrite what was just read and written
    __syncthreads();
    wk.advance(p, sg);
  }
}

template <typename T, int D, int NT>
int launch16(const CacheAttnParams& p, const CacheMaps& maps, cudaStream_t stream) {
  using L = Smem16<D, NT>;
  static bool attr_set[32] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 31]) {
    if (cudaFuncSetAttribute(cache_decode16_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal) != cudaSuccess) return TB200_ERR_CUDA;
    attr_set[dev & 31] = true;
  }
  return launch_decode_grid(cache_decode16_kernel<T, D, NT>, p, L::kTotal, stream, p, maps);
}

template <typename T>
int launch16(const CacheAttnParams& p, const CacheMaps& maps, int head_dim, int nt, cudaStream_t stream) {
  if (head_dim == 128) return nt == 1 ? launch16<T, 128, 1>(p, maps, stream) : launch16<T, 128, 2>(p, maps, stream);
  return nt == 1 ? launch16<T, 64, 1>(p, maps, stream) : launch16<T, 64, 2>(p, maps, stream);
}

}  // namespace

int cache16_stretches(int num_sms) { return 2 * num_sms; }   // two CTAs per SM: 97 KB of shared memory each

int launch_cache16(const CacheAttnParams& p, const tb200_cache_attn_args& a, int unit_rows, cudaStream_t stream) {
  const int nt = unit_rows / 8;
  CacheMaps maps;
  const uint64_t d = static_cast<uint64_t>(a.head_dim);
  const uint64_t dims[4] = {d, static_cast<uint64_t>(a.cache_len), static_cast<uint64_t>(a.n_kv_heads), static_cast<uint64_t>(a.batch)};
  const uint32_t box[4] = {64, kTile, 1, 1};
  auto map4 = [&](CUtensorMap* map, const void* base, const int64_t (&st)[3]) {   // strides: batch, head, row; unused ones get a valid value
    const uint64_t strides[3] = {a.cache_len > 1 ? static_cast<uint64_t>(st[2]) * 2 : d * 2, a.n_kv_heads > 1 ? static_cast<uint64_t>(st[1]) * 2 : d * 2,
                                 a.batch > 1 ? static_cast<uint64_t>(st[0]) * 2 : d * 2};
    return make_tensor_map(map, base, 4, dims, strides, box);
  };
  int status = map4(&maps.k, a.k_cache, a.k_stride);
  if (status == TB200_OK) status = map4(&maps.v, a.v_cache, a.v_stride);
  if (status != TB200_OK) return status;
  return a.dtype == TB200_BF16 ? launch16<__nv_bfloat16>(p, maps, a.head_dim, nt, stream) : launch16<__half>(p, maps, a.head_dim, nt, stream);
}

}  // namespace tb200
