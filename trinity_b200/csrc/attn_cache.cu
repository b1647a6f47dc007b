// Attention over a cache that already holds the new rows: tb200_attn_window (16-bit caches) and tb200_kv4_attn (4-bit
// caches), per-sequence lengths, an optional sliding window with a few first positions that stay visible.
//
// cache_decode_kernel: few query rows per sequence on a 4-bit cache (units, line and stretches: cache_line.cuh; a warp has
// its own ring of bulk copies, no CTA-wide barrier inside a segment).  Bound: HBM (the visible cache rows are read once per key/value
// head), and the instructions that turn 4-bit codes into matrix operands.
//
//   math     transposed: S^T = K Q^T (keys are the rows of the MMA, query rows its 8 columns), O^T = V^T P^T.
//   4 bits   a code c needs no conversion: the bits c in the low mantissa of an otherwise zero fp16 are the number
//            c * 2^-24, one nibble higher c * 2^-20, and the tensor core takes such (subnormal) numbers exactly.  One
//            AND per two codes makes an operand.  With K = lo + c s per group of 64:  q.k = sum_g s_g (q.c)_g + lo_g sum(q)_g,
//            so s and lo meet the scores in fp32 and no key is ever rounded.  With V:  o = sum_g [sum_j (p_j s_jg)(c_jd - 8) +
//            sum_j p_j (lo_jg + 8 s_jg)]: the scale goes into the probability (rounded to fp16, after a power of two per group
//            that brings the largest p s near 2^14), the second sum is fp32, and for fp16 outputs the 8 is taken out with the SAME
//            rounded probabilities (an MMA against a constant 8), so that the rounding error is that of centred codes, 2.6
//            times smaller; bf16 outputs are rounded sixteen times more coarsely than that and do without.
//            q is brought to fp16 by a power of two per row: inputs lose nothing within 2^-25 (bf16; fp16: 2^-22) of the row's
//            largest.
//   H = 2    four query rows or fewer (one token of up to four query heads per kv head): they fill half of the eight columns,
//            so columns 4 to 7 repeat them, and each column takes the probabilities of half the keys: a thread then has two
//            scores of sixteen keys to work on instead of four, and a row comes in two shares like those of two warps.
//   measured one token of 24 sequences of 1 to 16384 positions, 32/8 heads of 128, bf16: 52.4 us for 223 MB, 65 % of the copy
//            bandwidth; an instruction issues in half of the cycles, the tensor pipe is busy in a quarter of them: what is
//            left is the latency of each warp's chain scores -> maximum -> exponentials -> products, with the 8 to 12 warps
//            per SM that the registers allow.
#include <math.h>

#include <type_traits>

#include "cache_line.cuh"

namespace tb200 {

namespace {

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {   // d = a b
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// (s, lo) of a row's groups as floats
template <typename T, int NG> __device__ __forceinline__ void load_meta(const uint8_t* at, float2 (&m)[NG]) {
  if constexpr (NG == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(at);
    m[0] = Pack2<T>::unpack(u.x);
    m[1] = Pack2<T>::unpack(u.y);
  } else {
    m[0] = Pack2<T>::unpack(*reinterpret_cast<const uint32_t*>(at));
  }
}

// Tile (keys), stages of a warp's ring and CTAs per SM of an instance.  An unrolled tile of 64 keys gives the scheduler the
// most to interleave; with two column blocks at D = 128 its registers no longer fit and 32 keys are faster (42 against 60 us
// for five rows of 16 sequences), as 64 keys are elsewhere (24 long sequences: 55 against 59 us).
template <int D, int NT, int H> struct DecShape {
  static constexpr int kTile = D == 128 && NT == 2 ? 32 : 64, kStages = 2, kCtas = NT == 1 && (D == 64 || H == 2) ? 3 : 2;
};
template <int D, int NT, int H> struct DecSmem {
  static constexpr int kTile = DecShape<D, NT, H>::kTile, kStages = DecShape<D, NT, H>::kStages;
  static constexpr int kR = 8 * NT / H;                    // query rows of a unit
  static constexpr int kCodes = kTile * D / 2;             // bytes of one tile's codes
  static constexpr int kMeta = kTile * (D / 64) * 4;
  static constexpr int kStage = 2 * (kCodes + kMeta);      // K codes, V codes, K meta, V meta
  static constexpr int kRing = kStages * kStage;           // per warp
  static constexpr int kBarOff = kWarps * kRing;
  // the merge buffers take the place of the rings, which are empty by then
  static_assert(MergeSmem<D, NT>::kBytes <= kBarOff, "the merge buffers must fit where the rings were");
  static constexpr int kShareOff = kBarOff + kWarps * kStages * 8 + 16;
  static constexpr int kTotal = kShareOff + ShareSmem<D, kR>::kBytes;
};

template <typename T, int D, int NT, int H>
__global__ void __launch_bounds__(kThreads, DecShape<D, NT, H>::kCtas) cache_decode_kernel(const __grid_constant__ CacheAttnParams p) {
  using L = DecSmem<D, NT, H>;
  constexpr int KN = 2 / H;   // keys of sixteen whose scores a thread works on
  constexpr int NG = D / 64;
  constexpr int R = L::kR, kTile = L::kTile, kStages = L::kStages;
  // fp16 outputs are worth the centred codes (see above); bf16's own rounding is sixteen times coarser than what they gain
  constexpr bool kCentre = !IsBf16<T>::value;
  constexpr bool kGroupScale = NG > 1 || IsBf16<T>::value;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * L::kRing;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff) + warp * kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kBarOff + kWarps * kStages * 8);
  const AbortCtx ctx{p.err, abort_flag, p.wait_limit};
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[i], 1);
    if (warp == 0) *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();

  Walk wk;
  if (!wk.begin(p, kTile, R, kWarps)) return;
  uint32_t used = 0;    // tiles this warp has taken through its ring
  bool ok = true;

  for (; wk.x < wk.x_end;) {
    const Segment sg = wk.segment(p, kTile, R);
    const Seq& sq = wk.sq;
    const int b = sg.b, h = sg.h, rt = sg.rt, v0 = sg.v0, v1 = sg.v1, n_rows = sg.n_rows;
    const long long crow = (static_cast<long long>(b) * p.Hkv + h) * p.cache_len;
    const int copy_end = min(p.cache_len, max(4, (sq.n + 3) & ~3));   // cache rows worth copying: whole 16 bytes of meta

    // lanes 0 to 3 fetch a tile's K codes, V codes, K meta, V meta: each has its own source, row size and place
    const int what = lane & 3;
    const uint32_t row_bytes = what < 2 ? D / 2 : NG * 4;
    const uint8_t* src = (what == 0 ? p.k_codes : what == 1 ? p.v_codes : what == 2 ? p.k_meta : p.v_meta) + crow * row_bytes;
    uint8_t* dst = ring + (what & 1) * (what < 2 ? L::kCodes : L::kMeta) + (what < 2 ? 0 : 2 * L::kCodes);
    auto issue = [&](int v, uint32_t slot) {   // whole warp: tile v of the unit into ring slot `slot`
      const int k0 = wk.tile_of(v) * kTile;
      const uint32_t rows = static_cast<uint32_t>(min(kTile, copy_end - k0));
      if (lane == 0) mbar_arrive_expect_tx(&bars[slot], rows * (D + NG * 8));
      __syncwarp();
      if (lane < 4) bulk_load(dst + slot * L::kStage, src + static_cast<long long>(k0) * row_bytes, rows * row_bytes, &bars[slot]);
    };
    auto drain = [&](int v) {   // a wait gave up: the copies in flight (tile v and those behind it) get their time to land
      for (int i = 0; i < kStages && v + i * kWarps < v1; ++i) {
        const uint32_t u = used + i;
        const long long t0 = clock64();
        while (!mbar_try_wait(&bars[u % kStages], (u / kStages) & 1) && clock64() - t0 < p.wait_limit) {
        }
      }
    };
    if (ok) {
#pragma unroll
      for (int i = 0; i < kStages; ++i)
        if (v0 + warp + i * kWarps < v1) issue(v0 + warp + i * kWarps, (used + i) % kStages);
    }

    // ---- the unit's query rows: MMA column m is row rt * R + m, i.e. (token, query head of the group)
    uint32_t qf[NT][NG][4][2];
    float qs[NT][NG][2], cf[NT][2], up[NT], down[NT], sum[NT][NG];
    int cpos[NT][2];
    uint32_t unit_top = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int m = rt * R + (nt * 8 + g) % R;
      const bool live = m < n_rows;
      const int tok = live ? m / p.group : 0;
      const int hq = h * p.group + (live ? m - tok * p.group : 0);
      const T* qp = reinterpret_cast<const T*>(p.q) + b * p.qs[0] + hq * p.qs[1] + tok * p.qs[2] + t * 16;
      float v[NG][16];
      float top = 0.f;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 raw = live ? __ldg(reinterpret_cast<const uint4*>(qp + gr * 64) + i) : make_uint4(0u, 0u, 0u, 0u);
          const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = Pack2<T>::unpack(w[e]);
            v[gr][i * 8 + 2 * e] = f.x;
            v[gr][i * 8 + 2 * e + 1] = f.y;
          }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(v[gr][e]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      unit_top = max(unit_top, __float_as_uint(top));
      // a power of two that brings the row's largest magnitude to [2^14, 2^15): small ones keep their digits beside a large one
      const int ex = max(static_cast<int>(__float_as_uint(top) >> 23), 15);
      up[nt] = __uint_as_float(static_cast<uint32_t>(268 - ex) << 23);        // 2^(141 - ex)
      down[nt] = __uint_as_float(static_cast<uint32_t>(ex - 14) << 23);       // its inverse
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) x += v[gr][e] *= up[nt];
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        sum[nt][gr] = x + __shfl_xor_sync(0xffffffffu, x, 2);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const int e = (ks >> 1) * 8 + (ks & 1) * 2;
          qf[nt][gr][ks][0] = Pack2<__half>::pack(v[gr][e], v[gr][e + 4]);
          qf[nt][gr][ks][1] = Pack2<__half>::pack(v[gr][e + 1] * 0.0625f, v[gr][e + 5] * 0.0625f);
        }
      }
    }
    // The products come out times 2^-24.  Its inverse belongs to the row's factor cf, where large keys leave room for it; rows
    // from 2^64 on have none in cf and take it with s and lo (keys that would be too large for that have no finite score).
    const bool large = __reduce_max_sync(0xffffffffu, unit_top) >= (191u << 23);
    const float kf = large ? 16777216.f : 1.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {   // what columns 2t and 2t + 1 need of their rows
        const int src = (2 * t + c) * 4;
        // never 0 nor infinite: a hidden score is -inf times this, one of a key of zeros 0
        const float x = __shfl_sync(0xffffffffu, down[nt], src) * p.scale_log2 * (large ? 1.f : 16777216.f);
        cf[nt][c] = fminf(fmaxf(x, 1.17549435e-38f), 3.402823466e38f);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
          qs[nt][gr][c] = __shfl_sync(0xffffffffu, sum[nt][gr], src) * (large ? 1.f : 5.9604644775390625e-8f);   // 2^-24
        const int mc = rt * R + (nt * 8 + 2 * t + c) % R;
        cpos[nt][c] = mc < n_rows ? sq.n - sq.r + mc / p.group : -1;
      }

    // z, l: relative to 2^(maximum) and times 2^(5 - ev), o and o8 of a group times vf besides, see below
    float o[NT][NG][4][4], o8[NT][NG][2], z[NT][NG][2], l[NT][2], mx[NT][2], shift[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][gr][i][c] = o[nt][gr][i][2 + c] = 0.f;
          o8[nt][gr][c] = z[nt][gr][c] = 0.f;
        }
        mx[nt][c] = -INFINITY;
        l[nt][c] = shift[nt][c] = 0.f;
      }
    int ev = 60;   // biased exponent of the largest V scale so far, at least this
    // 2^(ev - exponent of the largest V scale so far of the group): groups of unlike size, and V below 2^(60 - 127) altogether,
    // bring p s near 2^14 all the same.  At most 2^120.  One group of fp16 needs none
    float vf[NG];
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) vf[gr] = kGroupScale ? 576460752303423488.f : 1.f;   // 2^59

    for (int v = v0 + warp; v < v1; v += kWarps) {
      const uint32_t slot = used % kStages;
      if (!ok || !mbar_wait(&bars[slot], (used / kStages) & 1, ctx, 701)) {   // (the CTA goes on to its barriers without this warp's keys)
        if (ok) drain(v);
        ok = false;
        break;
      }
      const uint8_t* st = ring + slot * L::kStage;
      const uint8_t* kc = st;
      const uint8_t* vc = st + L::kCodes;
      const uint8_t* km = st + 2 * L::kCodes;
      const uint8_t* vm = km + L::kMeta;
      const int k0 = wk.tile_of(v) * kTile;
      // every key of the tile visible to every row of the sequence?
      const bool full = k0 + kTile - 1 <= sq.n - sq.r && (p.window == 0 || k0 > sq.n - 1 - p.window || k0 + kTile - 1 < p.sinks);

      // A tile that every row sees altogether is one stretch of code without a branch (what the scheduler can interleave ends
      // at a branch: with the masks behind branches of their own, the loop took a fifth longer).
      auto tile = [&](auto whole_tile) {
        constexpr bool full = decltype(whole_tile)::value;
        // scores without the row's factor cf, then probabilities: rows 2t and 2t + 1, keys g and (H == 1) g + 8 of sixteen
        float s[kTile / 16][NT][2 * KN];
#pragma unroll
        for (int sp = 0; sp < kTile / 16; ++sp) {
          // MMA row (slot) 2a + e of eight is key a + 4 e: the four lanes of a column pair then read neighbouring rows
          const int key0 = sp * 16 + (g >> 1) + (g & 1) * 4, key1 = key0 + 8;
          float acc[NT][NG][4];
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            const uint2 w0 = *reinterpret_cast<const uint2*>(kc + key0 * (D / 2) + gr * 32 + t * 8);
            const uint2 w1 = *reinterpret_cast<const uint2*>(kc + key1 * (D / 2) + gr * 32 + t * 8);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              const uint32_t x0 = ((ks & 2) ? w0.y : w0.x) >> ((ks & 1) * 8), x1 = ((ks & 2) ? w1.y : w1.x) >> ((ks & 1) * 8);
              const uint32_t a0 = x0 & 0x000f000fu, a1 = x1 & 0x000f000fu, a2 = x0 & 0x00f000f0u, a3 = x1 & 0x00f000f0u;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                if (ks == 0) mma_f16_first(acc[nt][gr], a0, a1, a2, a3, qf[nt][gr][ks][0], qf[nt][gr][ks][1]);
                else mma_f16(acc[nt][gr], a0, a1, a2, a3, qf[nt][gr][ks][0], qf[nt][gr][ks][1]);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < KN; ++j) {
            const int key = H == 2 ? key0 + (t >> 1) * 8 : key0 + j * 8;
            float2 m[NG];
            load_meta<T, NG>(km + key * (NG * 4), m);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) m[gr].x *= kf;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float y = m[0].y * qs[nt][0][c];
                if constexpr (NG == 2) y = fmaf(m[1].y, qs[nt][1][c], y);
#pragma unroll
                for (int gr = 0; gr < NG; ++gr) y = fmaf(m[gr].x, H == 2 ? (t < 2 ? acc[nt][gr][c] : acc[nt][gr][2 + c]) : acc[nt][gr][2 * j + c], y);
                if (!full) {
                  const int a = k0 + key, pos = cpos[nt][c];
                  if (!(a <= pos && (p.window == 0 || a > pos - p.window || a < p.sinks))) y = -INFINITY;
                }
                s[sp][nt][2 * j + c] = y;
              }
          }
        }

        // ---- running maximum of the scores and of the V scales: what a thread sees of either decides whether the warp has
        //      to look closer
        auto scales = [&](auto take) {   // each lane two keys of 64: s and lo of their groups in V, as bits
#pragma unroll
          for (int i = 0; i < kTile / 32; ++i) {
            const int key = i * 32 + lane;
            bool alive = true;
            if (!full) {
              const int a = k0 + key;
              alive = a < sq.n && (p.window == 0 || a > sq.n - sq.r - p.window || a < p.sinks);
            }
            float2 mv[NG];
            load_meta<T, NG>(vm + key * (NG * 4), mv);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              const int u = __float_as_int(mv[gr].x), w = __float_as_int(fabsf(mv[gr].y));
              // lo counts where it is 2^60 times the scale: the sums of p lo have to stay in fp32 too
              if (alive && u < 0x7f800000 && w < 0x7f800000) take(gr, u, w - (60 << 23));
            }
          }
        };
        int big = 0;
        scales([&](int gr, int u, int w) { big = max(big, max(kGroupScale ? __float_as_int(__int_as_float(u) * vf[gr]) : u, w)); });
        float top[NT][2];
        bool grown = (big >> 23) > ev;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = s[0][nt][c];
#pragma unroll
            for (int sp = 0; sp < kTile / 16; ++sp)
#pragma unroll
              for (int j = 0; j < KN; ++j) x = fmaxf(x, s[sp][nt][2 * j + c]);
            top[nt][c] = x * cf[nt][c];
            grown |= top[nt][c] > mx[nt][c] + kSlack;
          }
        if (__any_sync(0xffffffffu, grown)) {
          [[maybe_unused]] int own[NG];
          if constexpr (kGroupScale) {   // (`big` may have passed the range of a float's bits)
            big = 0;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) own[gr] = 0;
            scales([&](int gr, int u, int w) {
              own[gr] = max(own[gr], u);
              big = max(big, max(u, w));
            });
          }
          const int ev_new = max(ev, __reduce_max_sync(0xffffffffu, big) >> 23);
          const float shrink = __uint_as_float(static_cast<uint32_t>(max(127 + ev - ev_new, 0)) << 23);   // 2^(ev - ev_new)
          float shrink_o[NG];
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            shrink_o[gr] = shrink;
            if constexpr (kGroupScale) {
              const int eg = ev + 127 - static_cast<int>(__float_as_uint(vf[gr]) >> 23);   // the group's exponent so far
              const int eg_new = max(max(eg, __reduce_max_sync(0xffffffffu, own[gr]) >> 23), ev_new - 120);
              shrink_o[gr] = __uint_as_float(static_cast<uint32_t>(max(127 + eg - eg_new, 0)) << 23);
              vf[gr] = __uint_as_float(static_cast<uint32_t>(127 + ev_new - eg_new) << 23);
            }
          }
          ev = ev_new;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float m_new = top[nt][c];
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, d));
              m_new = fmaxf(m_new, mx[nt][c]);
              const float e = m_new == -INFINITY ? 1.f : fast_exp2(mx[nt][c] - m_new), a = e * shrink;
              mx[nt][c] = m_new;
              shift[nt][c] = static_cast<float>(132 - ev) - (m_new == -INFINITY ? 0.f : m_new);   // 5 - (ev - 127): with p <= 2^kSlack, p s < 2^14
              l[nt][c] *= a;
#pragma unroll
              for (int gr = 0; gr < NG; ++gr) {
                z[nt][gr][c] *= a;
                const float ao = e * shrink_o[gr];
                if (kCentre) o8[nt][gr][c] *= ao;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  o[nt][gr][i][c] *= ao;
                  o[nt][gr][i][2 + c] *= ao;
                }
              }
            }
        }

#pragma unroll
        for (int sp = 0; sp < kTile / 16; ++sp)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int j = 0; j < KN; ++j) {
                s[sp][nt][2 * j + c] = fast_exp2(fmaf(s[sp][nt][2 * j + c], cf[nt][c], shift[nt][c]));
                l[nt][c] += s[sp][nt][2 * j + c];
              }
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          // a tile's products are summed from zero and then added in fp32: the tensor core's additions truncate, and over
          // thousands of keys with codes of one sign that would add up
          float part[NT][4][4];
          [[maybe_unused]] float part8[NT][4];
#pragma unroll
          for (int sp = 0; sp < kTile / 16; ++sp) {
            const int key0 = sp * 16 + (g >> 1) + (g & 1) * 4 + (H == 2 ? (t >> 1) * 8 : 0);
            float2 m[KN];
            float lo8[KN];
#pragma unroll
            for (int j = 0; j < KN; ++j) {
              m[j] = Pack2<T>::unpack(*reinterpret_cast<const uint32_t*>(vm + ((key0 + j * 8) * NG + gr) * 4));
              lo8[j] = kCentre ? fmaf(8.f, m[j].x, m[j].y) : m[j].y;
              if (kGroupScale) m[j].x *= vf[gr];
            }
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float w[2 * KN];
#pragma unroll
              for (int j = 0; j < KN; ++j)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  const float e = s[sp][nt][2 * j + c];
                  w[2 * j + c] = e * m[j].x;
                  if (full) z[nt][gr][c] = fmaf(e, lo8[j], z[nt][gr][c]);
                  // what a row does not see may hold anything: 0 * inf and 0 * NaN must not arise
                  else if (e > 0.f) z[nt][gr][c] = fmaf(e, lo8[j], z[nt][gr][c]);
                  else w[2 * j + c] = 0.f;
                }
              const uint32_t x = transpose8x8(Pack2<__half>::pack(w[0], w[1]));
              if constexpr (H == 2) {   // columns 0 to 3 take the keys 0 to 7 of sixteen, columns 4 to 7 the others
                pf[nt][0] = g < 4 ? x : 0u;
                pf[nt][1] = g < 4 ? 0u : x;
              } else {
                pf[nt][0] = x;
                pf[nt][1] = transpose8x8(Pack2<__half>::pack(w[2 * KN - 2], w[2 * KN - 1]));
              }
              if constexpr (kCentre) {
                if (sp == 0) mma_f16_first(part8[nt], 0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u, pf[nt][0], pf[nt][1]);
                else mma_f16(part8[nt], 0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u, pf[nt][0], pf[nt][1]);
              }
            }
            // MMA columns 2t, 2t+1 (and 2t+8, 2t+9) of V^T are keys t, t + 4 (and t + 8, t + 12); row g of the four row tiles
            // holds elements 8 g + {0, 2, 4, 6}, row g + 8 the odd ones
            const uint8_t* vp = vc + (sp * 16 + t) * (D / 2) + gr * 32 + g * 4;
            const uint32_t wa = *reinterpret_cast<const uint32_t*>(vp), wb = *reinterpret_cast<const uint32_t*>(vp + 4 * (D / 2));
            const uint32_t wc = *reinterpret_cast<const uint32_t*>(vp + 8 * (D / 2)), wd = *reinterpret_cast<const uint32_t*>(vp + 12 * (D / 2));
            const uint32_t xl = __byte_perm(wa, wb, 0x5410), xh = __byte_perm(wa, wb, 0x7632);
            const uint32_t yl = __byte_perm(wc, wd, 0x5410), yh = __byte_perm(wc, wd, 0x7632);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t x0 = ((i & 2) ? xh : xl) >> ((i & 1) * 8), y0 = ((i & 2) ? yh : yl) >> ((i & 1) * 8);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                if (sp == 0) mma_f16_first(part[nt][i], x0 & 0x000f000fu, x0 & 0x00f000f0u, y0 & 0x000f000fu, y0 & 0x00f000f0u, pf[nt][0], pf[nt][1]);
                else mma_f16(part[nt][i], x0 & 0x000f000fu, x0 & 0x00f000f0u, y0 & 0x000f000fu, y0 & 0x00f000f0u, pf[nt][0], pf[nt][1]);
              }
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              if constexpr (kCentre) o8[nt][gr][c] += part8[nt][c];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                o[nt][gr][i][c] += part[nt][i][c];
                o[nt][gr][i][2 + c] += part[nt][i][2 + c];
              }
            }
          }
        }
      };
      if (full) tile(std::true_type{});
      else tile(std::false_type{});
      __syncwarp();   // every lane has read the slot
      if (v + kStages * kWarps < v1) issue(v + kStages * kWarps, slot);
      ++used;
    }

    // ---- this warp's share of the segment into shared memory: o relative to its own maximum
    __syncthreads();   // every warp is done with its ring
    using M = MergeSmem<D, NT>;
    float* wm = reinterpret_cast<float*>(smem) + warp * M::kR * M::kPitch;
    float2* wml = reinterpret_cast<float2*>(smem + M::kMlOff) + warp * M::kR;
    const float fe = __uint_as_float(static_cast<uint32_t>(ev - 5) << 23);   // 2^(ev - 127 - 5): out of the accumulators' scale
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int m = nt * 8 + 2 * t + c;
        float ls = l[nt][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, d);
        if (g == 0) wml[m] = make_float2(mx[nt][c], ls * fe);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          float zs = z[nt][gr][c];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) zs += __shfl_xor_sync(0xffffffffu, zs, d);
          const float a8 = kCentre ? o8[nt][gr][c] : 0.f;
          const float out = __uint_as_float((278u << 23) - __float_as_uint(vf[gr]));   // 2^24 / vf
#pragma unroll
          for (int i = 0; i < 4; ++i)   // row g + 8 holds codes times 2^-20
            *reinterpret_cast<float2*>(wm + m * M::kPitch + gr * 64 + g * 8 + 2 * i) =
                make_float2(fmaf(o[nt][gr][i][c] - a8, out, zs) * fe, fmaf(o[nt][gr][i][2 + c] * 0.0625f - a8, out, zs) * fe);
        }
      }
    __syncthreads();
    merge_segment<T, D, NT, H>(p, smem, smem + L::kShareOff, wk, sg);
    fence_proxy_async_smem();   // the next bulk copies overwrite what was just read and written
    __syncthreads();
    wk.advance(p, sg);
  }
}

// Merges the partial results of the units that lie in several stretches.  CTA (x, y): rows y * kRows to y * kRows + kRows - 1
// of record x's unit.  The unit begins in stretch c; its first part is in slot 2c + 1, the others in the slots 2c' of the
// stretches c' it covers.  A group of D / 4 threads takes every kSteps-th part of a row, and the groups' sums are added in a
// fixed order.  One row per CTA where units have many parts (one sequence of 71 heads, 65536 positions, 99 parts a unit: 22 us
// for both kernels instead of 27 with four rows), else as many as make two groups a row.
constexpr int kCombineThreads = 128, kCombineAhead = 4;
template <typename T, int D, int R, int kRows>
__global__ void __launch_bounds__(kCombineThreads) cache_combine_kernel(const __grid_constant__ CacheAttnParams p) {
  constexpr int kLanes = D / 4, kGroups = kCombineThreads / kLanes, kSteps = kGroups / kRows;
  __shared__ float4 red[kGroups][kLanes];
  __shared__ float red_sum[kGroups];
  pdl_launch_dependents();
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int row = group % kRows, step = group / kRows;
  pdl_wait();
  const int4 rec = __ldcg(p.split + blockIdx.x);
  int b = rec.x, h = rec.y, rt = rec.z, c = blockIdx.x;
  if (p.record_per_unit) {
    const int bh = c / p.row_tiles;
    rt = c - bh * p.row_tiles;
    b = bh / p.Hkv;
    h = bh - b * p.Hkv;
    c = rec.x;
  }
  const int m = blockIdx.y * kRows + row, mr = rt * R + m;
  const int r = p.q_rows ? max(0, min(__ldg(p.q_rows + b), p.S)) : p.S;
  if (rt * R + static_cast<int>(blockIdx.y) * kRows >= r * p.group) return;   // (a unit without rows has left no record)
  const int parts = rec.w;
  if (parts == 0) return;
  auto slot = [&](int i) { return static_cast<long long>(2 * (c + i) + (i == 0 ? 1 : 0)) * R + m; };
  auto load = [&](int i, float4& v, float2& ml) {
    v = make_float4(0.f, 0.f, 0.f, 0.f);
    ml = make_float2(-INFINITY, 0.f);
    if (i < parts) {
      v = __ldcg(reinterpret_cast<const float4*>(p.part_o + slot(i) * D) + lane);
      ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + slot(i));
    }
  };
  float4 v[kCombineAhead];
  float2 ml[kCombineAhead];
#pragma unroll
  for (int k = 0; k < kCombineAhead; ++k) load(step + k * kSteps, v[k], ml[k]);
  float top = -INFINITY;
#pragma unroll 4
  for (int i = lane; i < parts; i += kLanes) top = fmaxf(top, __ldcg(p.part_ml + slot(i) * 2));
#pragma unroll
  for (int d = kLanes / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = step; i0 < parts; i0 += kCombineAhead * kSteps) {
#pragma unroll
    for (int k = 0; k < kCombineAhead; ++k) {
      const float f = ml[k].x == -INFINITY ? 0.f : fast_exp2(ml[k].x - top);
      sum = fmaf(f, ml[k].y, sum);
      acc.x = fmaf(f, v[k].x, acc.x); acc.y = fmaf(f, v[k].y, acc.y); acc.z = fmaf(f, v[k].z, acc.z); acc.w = fmaf(f, v[k].w, acc.w);
    }
#pragma unroll
    for (int k = 0; k < kCombineAhead; ++k) load(i0 + (kCombineAhead + k) * kSteps, v[k], ml[k]);
  }
  if constexpr (kSteps > 1) {
    red[group][lane] = acc;
    if (lane == 0) red_sum[group] = sum;
    __syncthreads();
    if (step > 0) return;
#pragma unroll
    for (int i = 1; i < kSteps; ++i) {
      const float4 a = red[i * kRows + row][lane];
      acc.x += a.x; acc.y += a.y; acc.z += a.z; acc.w += a.w;
      sum += red_sum[i * kRows + row];
    }
  }
  if (mr >= r * p.group) return;
  const float inv = sum > 0.f ? 1.f / sum : sum;   // 0: the row sees nothing; NaN stays
  const int tok = mr / p.group;
  T* op = reinterpret_cast<T*>(p.o) + b * p.os[0] + (h * p.group + mr - tok * p.group) * p.os[1] + tok * p.os[2] + lane * 4;
  *reinterpret_cast<uint2*>(op) = make_uint2(Pack2<T>::pack(acc.x * inv, acc.y * inv), Pack2<T>::pack(acc.z * inv, acc.w * inv));
}

int check_attn(const tb200_cache_attn_args* a, bool kv4) {
  if (a == nullptr) return TB200_ERR_INVALID;
  if (a->dtype != TB200_BF16 && a->dtype != TB200_F16) return TB200_ERR_UNSUPPORTED;
  if (a->head_dim != 64 && a->head_dim != 128) return TB200_ERR_UNSUPPORTED;
  if (a->batch < 0 || a->rows < 0 || a->n_kv_heads < 1 || a->n_q_heads < 1 || a->n_q_heads % a->n_kv_heads || a->cache_len < 1) return TB200_ERR_INVALID;
  if (a->batch > kMaxExtent || a->cache_len > kMaxExtent || static_cast<int64_t>(a->n_q_heads) * a->rows > kMaxExtent) return TB200_ERR_INVALID;
  if (a->window < 0 || a->sinks < 0 || !(a->sm_scale >= 1e-30f) || !(a->sm_scale <= 1e38f)) return TB200_ERR_INVALID;
  if (a->batch == 0 || a->rows == 0) return TB200_OK;   // nothing to read or write: empty tensors have no address
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

// Decode kernel or prompt kernel, by the query rows of a sequence that share a kv head (new tokens x query heads per kv head).
// 16 bits: the prompt kernel packs the rows into tiles of 128, the decode kernel reads the cache once per 16 rows.  16
// sequences of 2048 positions, 32/8 heads, decode and prompt kernel in us: 16 rows 34 / 37, 32 rows 37 / 37, 64 rows 62 / 37;
// one head per kv head 16 rows 34 / 37; 71 heads on one, a single token, 4 x 16384 positions: 21 / 21.
// 4 bits: the prompt kernel needs the visible rows in 16 bits first: 32 rows 40 / 65, 64 rows 68 / 66, 96 rows 97 / 66; 71
// heads, a single token 23 / 25.  A single token never takes that copy.
bool takes_prompt_kernel(int64_t rows, int tokens, bool kv4) { return kv4 ? rows > 64 && tokens > 1 : rows > 16; }

// Query rows of a unit: the smallest form that holds a sequence's rows of one kv head, else as many as there are.  Four rows:
// see H at cache_decode_kernel.  24 rows (4 bits, D = 64: with D = 128 the accumulators do not fit): a tile takes 4/3 of the
// instructions of one of 16 rows, for the codes become operands once for all columns, so it is taken where that saves a third
// of the units or so.  In us with 16 and 24 rows, fp16, one token: 4 sequences of 71 heads on one, 131072 positions
// 69 / 59, 65536 41 / 38; 16 sequences of 192 heads on 8, 16384 positions 102 / 78.
int unit_rows_for(int64_t rows, int head_dim, bool kv4) {
  if (kv4 && head_dim == 64 && (rows + 23) / 24 * 4 < (rows + 15) / 16 * 3) return 24;
  return kv4 && rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
}
int kv4_ctas(int head_dim, int unit_rows) {
  if (head_dim == 128) return unit_rows == 4 ? DecShape<128, 1, 2>::kCtas : unit_rows == 8 ? DecShape<128, 1, 1>::kCtas : DecShape<128, 2, 1>::kCtas;
  if (unit_rows == 24) return DecShape<64, 3, 1>::kCtas;
  return unit_rows == 4 ? DecShape<64, 1, 2>::kCtas : unit_rows == 8 ? DecShape<64, 1, 1>::kCtas : DecShape<64, 2, 1>::kCtas;
}

constexpr int kClusterKeys = 640;
constexpr size_t kCopyBytes = size_t{256} << 20, kCopyMost = size_t{1} << 30;

struct AttnPlan {
  bool prompt = false;       // the prompt kernel (attn2.cu), on a 4-bit cache after reading it back into the workspace
  int unit_rows = 8;         // decode: query rows of a unit
  int row_tiles = 1;         // units per (sequence, kv head) at most
  int cluster = 0;           // CTAs per unit, 0: the line
  int stretches = 0;
  int pack = 1, kv_splits = 1;   // prompt
  // prompt on 4 bits: positions and layout of the 16-bit copy (Kv4PromptOperands), and of how many sequences and kv heads it is at
  // a time.  What follows is the size of one such piece.
  int copy_len = 0, packed_head = -1, piece_seqs = 0, piece_heads = 0;
  size_t part_o = 0, part_ml = 0, split = 0;               // bytes
  size_t cache16 = 0, q16 = 0, q_factor = 0, head_factor = 0;   // prompt on 4 bits: one of the two caches; bf16: q and the factors
  // + what brings the caller's address up to a multiple of 256
  size_t total() const { return part_o == 0 && cache16 == 0 ? 0 : part_o + part_ml + split + 2 * cache16 + q16 + q_factor + head_factor + 256; }
};
// A window as long as the cache hides nothing; first positions matter only beside a window.
int window_of(const tb200_cache_attn_args* a) { return a->window < a->cache_len ? a->window : 0; }
int sinks_of(const tb200_cache_attn_args* a) { return window_of(a) > 0 ? (a->sinks < a->cache_len ? a->sinks : a->cache_len) : 0; }

AttnPlan plan_attn(const tb200_cache_attn_args* a, bool kv4, int num_sms) {
  AttnPlan pl;
  const int window = window_of(a), sinks = sinks_of(a);
  const int64_t rows = static_cast<int64_t>(a->rows) * (a->n_q_heads / a->n_kv_heads);
  pl.prompt = takes_prompt_kernel(rows, a->rows, kv4);
  if (pl.prompt) {
    const int64_t seen = window > 0 ? static_cast<int64_t>(window) + a->rows + sinks : a->cache_len;
    pl.pack = attn_seq_pack(a->rows, a->n_q_heads, a->n_kv_heads, a->cache_len, window, sinks);
    pl.piece_seqs = a->batch;
    pl.piece_heads = a->n_kv_heads;
    if (kv4) {
      // The copy holds what a sequence can see, and a piece of the call at a time where it would be larger than kCopyBytes: a
      // cache is held in 4 bits where 16 do not fit.  Up to kCopyMost where a piece would have fewer than two items per SM, with
      // the keys in 16 shares; one (sequence, kv head) is the least.  32/8 heads of 128, bf16, the whole cache copied against
      // this, MiB of scratch and us: 24 sequences of 16384 and 20 tokens 1540, 791 / 262, 790; 100 tokens 1556, 1115 / 272, 1251;
      // 500 tokens 1632, 3170 / 272, 3490; 16 sequences of 131072 and 20 tokens 8195, 3700 / 1030, 4160; under a window of 1000
      // 8195, 411 / 67, 48.
      const int64_t head = (static_cast<int64_t>(sinks) + 15) & ~15;
      const int64_t packed = head + window + a->rows;
      pl.copy_len = a->cache_len;
      if (window > 0 && packed < a->cache_len) {
        pl.copy_len = static_cast<int>(packed);
        pl.packed_head = static_cast<int>(head);
      }
      const size_t one = static_cast<size_t>(pl.copy_len) * a->head_dim * 4;   // K and V
      const int group = a->n_q_heads / a->n_kv_heads, tokens = 2 * (128 / pl.pack);
      const size_t items = static_cast<size_t>(group / pl.pack) * ((a->rows + tokens - 1) / tokens);   // of a (sequence, kv head)
      const size_t busy = 2 * num_sms / (items * 16), most = kCopyMost / one;
      size_t fit = busy < most ? busy : most;
      if (fit < kCopyBytes / one) fit = kCopyBytes / one;
      if (fit < 1) fit = 1;
      if (fit < static_cast<size_t>(a->n_kv_heads)) {
        const int parts = static_cast<int>((a->n_kv_heads + fit - 1) / fit);
        pl.piece_seqs = 1;
        pl.piece_heads = (a->n_kv_heads + parts - 1) / parts;
      } else if (fit / a->n_kv_heads < static_cast<size_t>(a->batch)) {
        const int seqs = static_cast<int>(fit / a->n_kv_heads), parts = (a->batch + seqs - 1) / seqs;
        pl.piece_seqs = (a->batch + parts - 1) / parts;
      }
    }
    const int q_heads = a->n_q_heads / a->n_kv_heads * pl.piece_heads;
    // the splits count blocks of 256 rows: tokens times packed heads
    pl.kv_splits = attn_kv_splits(pl.piece_seqs, (a->rows + 128 / pl.pack - 1) / (128 / pl.pack) * 128, q_heads / pl.pack,
                                  static_cast<int>(seen < a->cache_len ? seen : a->cache_len), num_sms);
    if (pl.kv_splits > 1) {
      const size_t prows = static_cast<size_t>(pl.kv_splits) * pl.piece_seqs * q_heads * a->rows;
      pl.part_o = align_up(prows * a->head_dim * sizeof(float), 256);
      pl.part_ml = align_up(prows * 2 * sizeof(float), 256);
    }
    if (kv4) pl.cache16 = align_up(static_cast<size_t>(pl.piece_seqs) * pl.piece_heads * pl.copy_len * a->head_dim * 2, 256);
    if (kv4 && a->dtype == TB200_BF16) {
      const size_t q_rows = static_cast<size_t>(pl.piece_seqs) * q_heads * a->rows;
      pl.q16 = align_up(q_rows * a->head_dim * 2, 256);
      pl.q_factor = align_up(q_rows * sizeof(float), 256);
      pl.head_factor = align_up(static_cast<size_t>(pl.piece_seqs) * pl.piece_heads * 4 * sizeof(float), 256);
    }
    return pl;
  }
  const int64_t keys = window > 0 && static_cast<int64_t>(window) + a->rows + sinks < a->cache_len ? static_cast<int64_t>(window) + a->rows + sinks : a->cache_len;
  int ctas = 0, cluster = 1;
  int64_t units = 0;
  auto deal = [&](int unit_rows) {
    pl.unit_rows = unit_rows;
    pl.row_tiles = static_cast<int>((rows + unit_rows - 1) / unit_rows);
    ctas = kv4 ? num_sms * kv4_ctas(a->head_dim, unit_rows) : cache16_stretches(num_sms);
    units = static_cast<int64_t>(a->batch) * a->n_kv_heads * pl.row_tiles;
    for (cluster = 1; cluster < 8 && units * cluster * 2 <= ctas;) cluster *= 2;
    return units <= ctas && keys <= static_cast<int64_t>(kClusterKeys) * kWarps * cluster;
  };
  // A cluster per unit where the CTAs that are resident at a time give every warp kClusterKeys keys or fewer: one launch, no
  // partial results through HBM.  With more keys the line is safer, which does not care how long each sequence is.  Token on
  // 4 bits, 16 sequences of 32/8 heads, line and clusters in us: 2048 positions each 20.6 / 16.3, 4096 28.6 / 22.6; up to 8192
  // of different lengths 30.9 / 34.9 (1280 keys a warp).
  bool clusters = deal(unit_rows_for(rows, a->head_dim, kv4));
  // fewer units than the SMs hold in the largest clusters: 16 rows use more SMs (4 sequences of 71 heads, 2048 positions: 8.1
  // against 9.3 us)
  if (pl.unit_rows == 24 && clusters && cluster == 8) clusters = deal(16) || deal(24);
  if (clusters) {
    pl.cluster = cluster;
    pl.stretches = static_cast<int>(units * cluster);
    return pl;
  }
  pl.stretches = ctas;
  pl.part_o = align_up(static_cast<size_t>(pl.stretches) * 2 * pl.unit_rows * a->head_dim * sizeof(float), 256);
  pl.part_ml = align_up(static_cast<size_t>(pl.stretches) * 2 * pl.unit_rows * 2 * sizeof(float), 256);
  pl.split = align_up(static_cast<size_t>(pl.stretches) * sizeof(int4), 256);
  return pl;
}

CacheAttnParams make_params(const tb200_cache_attn_args* a, const DeviceState* st) {
  CacheAttnParams p;
  memset(&p, 0, sizeof(p));
  p.B = a->batch; p.S = a->rows; p.Hq = a->n_q_heads; p.Hkv = a->n_kv_heads; p.group = a->n_q_heads / a->n_kv_heads;
  p.cache_len = a->cache_len;
  p.window = window_of(a);
  p.sinks = sinks_of(a);
  p.scale_log2 = a->sm_scale * kLog2e;
  p.q = static_cast<const uint8_t*>(a->q);
  p.o = static_cast<uint8_t*>(a->o);
  for (int i = 0; i < 3; ++i) { p.qs[i] = a->q_stride[i]; p.os[i] = a->o_stride[i]; }
  p.kv_lens = a->kv_lens; p.q_rows = a->q_rows;
  p.k_codes = static_cast<const uint8_t*>(a->k_codes);
  p.v_codes = static_cast<const uint8_t*>(a->v_codes);
  p.k_meta = static_cast<const uint8_t*>(a->k_meta);
  p.v_meta = static_cast<const uint8_t*>(a->v_meta);
  p.err = st->err_word;
  p.wait_limit = wait_limit_cycles();
  return p;
}

template <typename T, int D, int NT, int H>
int launch_decode(const CacheAttnParams& p, cudaStream_t stream) {
  using L = DecSmem<D, NT, H>;
  static bool attr_set[32] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 31]) {
    if (cudaFuncSetAttribute(cache_decode_kernel<T, D, NT, H>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal) != cudaSuccess)
      return TB200_ERR_CUDA;
    attr_set[dev & 31] = true;
  }
  return launch_decode_grid(cache_decode_kernel<T, D, NT, H>, p, L::kTotal, stream, p);
}
template <typename T, int D>
int run_kv4(const CacheAttnParams& p, int unit_rows, cudaStream_t stream) {
  if (unit_rows == 4) return launch_decode<T, D, 1, 2>(p, stream);
  if constexpr (D == 64) {
    if (unit_rows == 24) return launch_decode<T, D, 3, 1>(p, stream);
  }
  return unit_rows == 8 ? launch_decode<T, D, 1, 1>(p, stream) : launch_decode<T, D, 2, 1>(p, stream);
}
template <typename T>
int run_kv4(const CacheAttnParams& p, int head_dim, int unit_rows, cudaStream_t stream) {
  return head_dim == 128 ? run_kv4<T, 128>(p, unit_rows, stream) : run_kv4<T, 64>(p, unit_rows, stream);
}

template <typename T, int D, int R>
int launch_combine(const CacheAttnParams& p, cudaStream_t stream) {
  constexpr int kRows = 256 / D;
  const unsigned records = static_cast<unsigned>(p.record_per_unit ? p.B * p.Hkv * p.row_tiles : p.stretches);
  const cudaError_t e = records * 16 <= static_cast<unsigned>(p.stretches)
                            ? launch_chained(cache_combine_kernel<T, D, R, 1>, dim3(records, R), dim3(kCombineThreads), 0, stream, p)
                            : launch_chained(cache_combine_kernel<T, D, R, kRows>, dim3(records, R / kRows), dim3(kCombineThreads), 0, stream, p);
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? TB200_OK : TB200_ERR_CUDA;
}
template <typename T, int D>
int launch_combine(const CacheAttnParams& p, int unit_rows, cudaStream_t stream) {
  if (unit_rows == 4) return launch_combine<T, D, 4>(p, stream);
  if constexpr (D == 64) {
    if (unit_rows == 24) return launch_combine<T, D, 24>(p, stream);
  }
  return unit_rows == 8 ? launch_combine<T, D, 8>(p, stream) : launch_combine<T, D, 16>(p, stream);
}
template <typename T>
int launch_combine(const CacheAttnParams& p, int head_dim, int unit_rows, cudaStream_t stream) {
  return head_dim == 128 ? launch_combine<T, 128>(p, unit_rows, stream) : launch_combine<T, 64>(p, unit_rows, stream);
}

int run_prompt(const tb200_cache_attn_args* a, bool kv4, const AttnPlan& pl, const CacheAttnParams& p, uint8_t* ws, int num_sms, cudaStream_t stream) {
  ChainScope chain;
  AttnSeqLaunch s;
  s.dtype = a->dtype;
  s.B = a->batch; s.S = a->rows; s.Hq = a->n_q_heads; s.Hkv = a->n_kv_heads; s.D = a->head_dim; s.cache_len = s.len = a->cache_len;
  s.window = p.window; s.sinks = p.sinks;
  s.sm_scale = a->sm_scale;
  s.q = a->q; s.o = a->o;
  s.kv_lens = a->kv_lens; s.q_rows = a->q_rows;
  s.pack = pl.pack;
  s.kv_splits = pl.kv_splits;
  s.part_o = reinterpret_cast<float*>(ws);
  s.part_ml = reinterpret_cast<float*>(ws + pl.part_o);
  s.k_cache = a->k_cache; s.v_cache = a->v_cache;
  for (int i = 0; i < 3; ++i) { s.q_stride[i] = a->q_stride[i]; s.o_stride[i] = a->o_stride[i]; s.k_stride[i] = a->k_stride[i]; s.v_stride[i] = a->v_stride[i]; }
  if (kv4) {
    Kv4PromptOperands to;
    uint8_t* at = ws + pl.part_o + pl.part_ml;
    to.len = s.len = pl.copy_len;
    to.packed_head = s.packed_head = pl.packed_head;
    to.k16 = at;
    to.v16 = at += pl.cache16;
    at += pl.cache16;
    if (a->dtype == TB200_BF16) {
      to.q16 = at;
      to.q_factor = reinterpret_cast<float*>(at += pl.q16);
      to.head_factor = reinterpret_cast<float*>(at += pl.q_factor);
      s.q = to.q16;
      s.q_factor = to.q_factor;
      s.head_factor = to.head_factor;
      s.q_stride[2] = a->head_dim;
      s.q_stride[1] = static_cast<int64_t>(a->rows) * a->head_dim;
      s.q_stride[0] = s.q_stride[1] * a->n_q_heads;
    }
    const int status = launch_kv4_prompt_operands(*a, p.window, p.sinks, to, num_sms, stream);
    if (status != TB200_OK) return status;
    s.k_cache = to.k16; s.v_cache = to.v16;
    s.k_stride[2] = s.v_stride[2] = a->head_dim;
    s.k_stride[1] = s.v_stride[1] = static_cast<int64_t>(pl.copy_len) * a->head_dim;
    s.k_stride[0] = s.v_stride[0] = s.k_stride[1] * a->n_kv_heads;
  }
  return launch_attn_fwd_seq(s, stream);
}

// A prompt on a 4-bit cache, piece by piece.  Each piece is a chain of its own: its first launch waits for the piece before,
// whose copy it overwrites.
int run_pieces(const tb200_cache_attn_args* a, const AttnPlan& pl, const CacheAttnParams& p, uint8_t* ws, int num_sms, cudaStream_t stream) {
  const int group = a->n_q_heads / a->n_kv_heads;
  for (int b0 = 0; b0 < a->batch; b0 += pl.piece_seqs)
    for (int h0 = 0; h0 < a->n_kv_heads; h0 += pl.piece_heads) {
      tb200_cache_attn_args x = *a;
      x.batch = a->batch - b0 < pl.piece_seqs ? a->batch - b0 : pl.piece_seqs;
      x.n_kv_heads = a->n_kv_heads - h0 < pl.piece_heads ? a->n_kv_heads - h0 : pl.piece_heads;
      x.n_q_heads = x.n_kv_heads * group;
      x.q = static_cast<const uint8_t*>(a->q) + 2 * (b0 * a->q_stride[0] + static_cast<int64_t>(h0) * group * a->q_stride[1]);
      x.o = static_cast<uint8_t*>(a->o) + 2 * (b0 * a->o_stride[0] + static_cast<int64_t>(h0) * group * a->o_stride[1]);
      x.kv_lens = a->kv_lens + b0;
      if (a->q_rows) x.q_rows = a->q_rows + b0;
      const int64_t crow = (static_cast<int64_t>(b0) * a->n_kv_heads + h0) * a->cache_len;   // (fewer heads: of one sequence)
      x.k_codes = static_cast<const uint8_t*>(a->k_codes) + crow * (a->head_dim / 2);
      x.v_codes = static_cast<const uint8_t*>(a->v_codes) + crow * (a->head_dim / 2);
      x.k_meta = static_cast<const uint8_t*>(a->k_meta) + crow * (a->head_dim / 16);
      x.v_meta = static_cast<const uint8_t*>(a->v_meta) + crow * (a->head_dim / 16);
      const int status = run_prompt(&x, true, pl, p, ws, num_sms, stream);
      if (status != TB200_OK) return status;
    }
  return TB200_OK;
}

int run_attn(const tb200_cache_attn_args* a, bool kv4, void* stream_) {
  const int bad = check_attn(a, kv4);
  if (bad != TB200_OK) return bad;
  int status = TB200_OK;
  DeviceState* st = device_state(&status);
  if (!st) return status;
  if (a->batch == 0 || a->rows == 0) return TB200_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  CacheAttnParams p = make_params(a, st);
  const AttnPlan pl = plan_attn(a, kv4, st->num_sms);
  if (pl.total() > 0 && (!a->workspace || a->workspace_bytes < pl.total())) return TB200_ERR_WORKSPACE;
  uint8_t* ws = reinterpret_cast<uint8_t*>(align_up(reinterpret_cast<size_t>(a->workspace), 256));
  if (pl.prompt) return kv4 ? run_pieces(a, pl, p, ws, st->num_sms, stream) : run_prompt(a, false, pl, p, ws, st->num_sms, stream);
  ChainScope chain;
  p.stretches = pl.stretches;
  p.record_per_unit = static_cast<int64_t>(a->batch) * a->n_kv_heads * pl.row_tiles <= pl.stretches;
  p.row_tiles = pl.row_tiles;
  p.cluster = pl.cluster;
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + pl.part_o);
  p.split = reinterpret_cast<int4*>(ws + pl.part_o + pl.part_ml);
  // positions on the line of tiles are 32-bit numbers
  const int64_t rows = static_cast<int64_t>(a->rows) * p.group;
  if ((rows / pl.unit_rows + 1) * a->n_kv_heads * a->batch * static_cast<double>(a->cache_len / 16 + 2) >= 2147483648.0) return TB200_ERR_UNSUPPORTED;
  if (!kv4) status = launch_cache16(p, *a, pl.unit_rows, stream);
  else if (a->dtype == TB200_BF16) status = run_kv4<__nv_bfloat16>(p, a->head_dim, pl.unit_rows, stream);
  else status = run_kv4<__half>(p, a->head_dim, pl.unit_rows, stream);
  if (status != TB200_OK || pl.cluster > 0) return status;
  return launch_cache_combine(p, a->dtype, a->head_dim, pl.unit_rows, stream);
}

size_t workspace_bytes(const tb200_cache_attn_args* a, bool kv4) {
  int status = TB200_OK;
  DeviceState* st = device_state(&status);
  if (!st || check_attn(a, kv4) != TB200_OK || a->batch == 0 || a->rows == 0) return 0;
  return plan_attn(a, kv4, st->num_sms).total();
}

}  // namespace

int launch_cache_combine(const CacheAttnParams& p, int dtype, int head_dim, int unit_rows, cudaStream_t stream) {
  return dtype == TB200_BF16 ? launch_combine<__nv_bfloat16>(p, head_dim, unit_rows, stream) : launch_combine<__half>(p, head_dim, unit_rows, stream);
}

}  // namespace tb200

using namespace tb200;

extern "C" {

int tb200_attn_window_check(const tb200_cache_attn_args* a) { return check_attn(a, false); }
int tb200_kv4_attn_check(const tb200_cache_attn_args* a) { return check_attn(a, true); }
size_t tb200_attn_window_workspace_bytes(const tb200_cache_attn_args* a) { return workspace_bytes(a, false); }
size_t tb200_kv4_attn_workspace_bytes(const tb200_cache_attn_args* a) { return workspace_bytes(a, true); }
int tb200_attn_window(const tb200_cache_attn_args* a, void* stream) { return run_attn(a, false, stream); }
int tb200_kv4_attn(const tb200_cache_attn_args* a, void* stream) { return run_attn(a, true, stream); }

}  // extern "C"
