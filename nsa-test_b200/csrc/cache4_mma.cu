// Attention over the 4-bit paged cache for few rows a request (decode, drafted tokens, selected blocks): bf16 queries on mma.m16n8k16 with
// fp16 operands and 32-bit sums.  How the work is cut up: cache4_attn.cuh.
//
// A block of four warps has 16 rows of a kv group; a warp takes half a page (32 keys) at a time, brought in by one bulk copy, with a running
// maximum, sum and output of its own; the warps' results are merged at the end of a segment.  The cache's layout is the products' B
// fragment, so a chunk's codes come with one 8-byte load per lane.
//
// Logits: a nibble c masked out of its word where it lies is the fp16 number c 2^-24 (or 16 c 2^-24: the bits of a number below 2^-13 are its
// multiple of 2^-24), so unpacking costs one AND per two codes; the sums start from -8 sum(q) 2^-24, which turns codes into values.  Each 32
// dimensions are multiplied by their scale in 32 bits.  Queries are scaled to a largest magnitude in [2^14, 2^15) per row (a power of two;
// bf16 has 8 bits, fp16 11, so only elements 2^-20 below the row's largest lose any) and the pairs whose codes arrive 16 times too large are
// divided by 16.  All of it is exact but for the 32-bit sums.
// Outputs: values times scales are exact in fp16; probabilities are rounded to fp16 (2^-11, an eighth of the output's own rounding).
// The reference maximum moves only when a row's maximum outgrows it by 2^8, so probabilities stay far below 65504.
//
// Bound by issue slots: about 380 instructions per 16 keys and warp, of which 40 products; HBM would take 126 clocks of an SM for them.
#include <algorithm>

#include "attn_args.cuh"
#include "cache4_attn.cuh"
#include "fa_sm100.cuh"
#include "sm100_ptx.cuh"

namespace nsa {

using namespace ptx;

constexpr int kMmThreads = 128, kMmWarps = 4, kMmRows = 16;
constexpr int kMmStages = 3;                         // half pages in flight per warp
constexpr int kMmKeys = 2 * kRecTokens;
constexpr int kMmOver = 1;                           // see Walk
constexpr float kMmGrow = 8.f;                       // log2 units

template <int GK, int GV>
struct MmaSmem {
  static constexpr int kRecBytes = (GK + GV) * kRecBytesPerGroup, kStageBytes = 2 * kRecBytes, kRingBytes = kMmWarps * kMmStages * kStageBytes;
  static constexpr int oQ = kRingBytes, oC = oQ + GK * 1024, kDynamic = oC + GK * 128;
  static constexpr int kBlocksPerSm = GV > 2 ? 3 : 5;
  static_assert(kMmWarps * kMmRows * GV * 32 * 4 <= kRingBytes, "the warps' results are merged in the ring");
  static_assert(4096 * 4 <= kRingBytes, "the requests' units are held in the ring");
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& x, uint32_t b0, uint32_t b1, const float4& c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y), "f"(c.z), "f"(c.w));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint4& x, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t code_bits(uint32_t x, uint32_t mask) {      // (x & mask) | 1024 in both halves
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, 0x64006400, 0xEA;" : "=r"(r) : "r"(x), "r"(mask));
  return r;
}

// what a warp keeps of a segment; the lane holds rows n and n + 8
template <int GV>
struct MmaState {
  float o[GV][4][4];
  float m[2], lim[2], top[2], l[2], c2[2], cl[2];      // lim: what a maximum has to exceed for m to move; c2, cl: a unit of the sums in log2 and natural logits
  int pos[2];
};

// The segment's queries: fragments into shared memory (warp w writes every fourth group), the rows' constants into registers.
template <int GK, int GV>
__device__ __forceinline__ void load_rows(const Cache4Args& a, const Segment& s, uint8_t* sq, float4* sc, MmaState<GV>& st) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, j = lane & 3;
  uint32_t frag[GK][2][4];
  float sum[GK][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = n + 8 * h, f = s.row0 + i;
    const bool row = i < s.nrows;
    st.pos[h] = row ? s.pos0 + f / a.hpg : -1;
    uint4 raw[GK];
    const __nv_bfloat16* src = (const __nv_bfloat16*)a.q + (s.tok0 + f / a.hpg) * a.sq_tok + (s.g * a.hpg + f % a.hpg) * a.sq_head + 8 * j;
    uint32_t mx = 0;
#pragma unroll
    for (int g = 0; g < GK; ++g) raw[g] = row ? *reinterpret_cast<const uint4*>(src + g * kGroupDims) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int g = 0; g < GK; ++g) {
      const uint32_t u[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = max(mx, max(u[e] & 0x7fffu, u[e] >> 16 & 0x7fffu));
    }
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const int k = mx ? min(14 - ((int)(mx >> 7) - 127), 100) : 0;
    // the scale's sign goes into the row, so that a larger sum is always the larger logit; scale 0 is a row of zeros
    const float up = __uint_as_float((uint32_t)(k + 127) << 23) * (a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : 0.f);
    st.cl[h] = (a.scale == 0.f ? 1.f : fabsf(a.scale)) * __uint_as_float((uint32_t)(127 - k) << 23) * 16777216.f;
    st.c2[h] = st.cl[h] * kLog2e;
#pragma unroll
    for (int g = 0; g < GK; ++g) {
      const uint32_t u[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
      float x[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(u[e] << 16) * up;
        x[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u) * up;
      }
      sum[g][h] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {                                 // dimensions e and e + 4: nibbles e, e + 4
        const float w = e & 1 ? 0.0625f : 1.f;
        const __half2 p = __floats2half2_rn(x[e] * w, x[e + 4] * w);
        sum[g][h] += (__low2float(p) + __high2float(p)) * (e & 1 ? 16.f : 1.f);
        frag[g][e >> 1][2 * (e & 1) + h] = as_u32(p);
      }
      sum[g][h] += __shfl_xor_sync(0xffffffffu, sum[g][h], 1);
      sum[g][h] += __shfl_xor_sync(0xffffffffu, sum[g][h], 2);
    }
    st.m[h] = st.lim[h] = st.top[h] = -CUDART_INF_F;
    st.l[h] = 0.f;
  }
#pragma unroll
  for (int g = 0; g < GK; ++g)
    if ((g & 3) == warp) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<uint4*>(sq + (g * 2 + e) * 512 + lane * 16) = make_uint4(frag[g][e][0], frag[g][e][1], frag[g][e][2], frag[g][e][3]);
      const float c = -4.76837158203125e-07f;                       // -8 * 2^-24
      if (j == 0) sc[g * 8 + n] = make_float4(sum[g][0] * c, sum[g][0] * c, sum[g][1] * c, sum[g][1] * c);
    }
#pragma unroll
  for (int g = 0; g < GV; ++g)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) st.o[g][e][i] = 0.f;
}

// 32 keys from position `base` on
template <int GK, int GV>
__device__ __forceinline__ void half_page(const Cache4Args& a, const Segment& s, const uint8_t* rec0, const uint8_t* sq, const float4* sc, int base, int minpos,
                                          int maxpos, int minlow, MmaState<GV>& st) {
  constexpr int kRecBytes = (GK + GV) * kRecBytesPerGroup;
  const int lane = threadIdx.x & 31, j = lane & 3;
  const uint8_t* codes = rec0 + lane * 8;
  const uint8_t* scales = rec0 + (GK + GV) * kChunkBytes + j * 8;
  float x[4][4];                  // [tile of 8 keys][row n: keys 2 j, 2 j + 1; row n + 8: the same]
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i >> 2][i & 3] = 0.f;
#pragma unroll
  for (int g = 0; g < GK; ++g) {
    const uint4 q0 = *reinterpret_cast<const uint4*>(sq + g * 1024 + lane * 16), q1 = *reinterpret_cast<const uint4*>(sq + g * 1024 + 512 + lane * 16);
    const float4 c0 = sc[g * 8 + (lane >> 2)];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint2 w = *reinterpret_cast<const uint2*>(codes + r * kRecBytes + g * kChunkBytes);
      const uint2 f2 = *reinterpret_cast<const uint2*>(scales + r * kRecBytes + g * kChunkScaleBytes);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t u = t ? w.y : w.x, v = u >> 8;
        float c[4];
        mma16816(c, q0, u & 0x000f000fu, u & 0x00f000f0u, c0);
        mma16816(c, q1, v & 0x000f000fu, v & 0x00f000f0u);
        const float2 f = __half22float2(as_half2(t ? f2.y : f2.x));
        float(&y)[4] = x[2 * r + t];
        y[0] = fmaf(c[0], f.x, y[0]);
        y[1] = fmaf(c[1], f.y, y[1]);
        y[2] = fmaf(c[2], f.x, y[2]);
        y[3] = fmaf(c[3], f.y, y[3]);
      }
    }
  }
  if (base + kMmKeys - 1 > minpos || (a.window > 0 && base <= maxpos - a.window)) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = base + 8 * t + 2 * j + (i & 1), p = st.pos[i >> 1];
        if (at > p || (a.window > 0 && at <= p - a.window)) x[t][i] = -CUDART_INF_F;
      }
  }
  float mx[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    mx[h] = fmaxf(fmaxf(fmaxf(x[0][2 * h], x[0][2 * h + 1]), fmaxf(x[1][2 * h], x[1][2 * h + 1])),
                  fmaxf(fmaxf(x[2][2 * h], x[2][2 * h + 1]), fmaxf(x[3][2 * h], x[3][2 * h + 1])));
    st.top[h] = fmaxf(st.top[h], mx[h]);
  }
  if (__any_sync(0xffffffffu, mx[0] > st.lim[0] || mx[1] > st.lim[1])) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float w = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 2));
      if (w > st.lim[h]) {
        const float f = ex2((st.m[h] - w) * st.c2[h]);
        st.m[h] = w;
        st.lim[h] = w + kMmGrow / st.c2[h];
        st.l[h] *= f;
#pragma unroll
        for (int g = 0; g < GV; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            st.o[g][e][2 * h] *= f;
            st.o[g][e][2 * h + 1] *= f;
          }
      }
    }
  }
  float b[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) b[h] = st.m[h] == -CUDART_INF_F ? 0.f : -st.m[h] * st.c2[h];
  uint32_t p[4][2];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float p0 = ex2(fmaf(x[t][2 * h], st.c2[h], b[h])), p1 = ex2(fmaf(x[t][2 * h + 1], st.c2[h], b[h]));
      st.l[h] += p0 + p1;
      p[t][h] = as_u32(__floats2half2_rn(p0, p1));
    }
  // what no row sees may never have been written: nothing of it enters, not as 0 times it either
  uint32_t keep[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
  if (base + kMmKeys - 1 > maxpos || base < minlow) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int at = base + 8 * t + 2 * j;
      keep[t] = (at <= maxpos && at >= minlow ? 0xffffu : 0u) | (at + 1 <= maxpos && at + 1 >= minlow ? 0xffff0000u : 0u);
    }
  }
  const __half2 bias = __float2half2_rn(-1032.f), sixteenth = __float2half2_rn(0.0625f), bias16 = __float2half2_rn(-72.f);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint4 pa = make_uint4(p[2 * r][0], p[2 * r][1], p[2 * r + 1][0], p[2 * r + 1][1]);
#pragma unroll
    for (int g = 0; g < GV; ++g) {
      const uint2 w = *reinterpret_cast<const uint2*>(codes + r * kRecBytes + (GK + g) * kChunkBytes);
      const uint2 f2 = *reinterpret_cast<const uint2*>(scales + r * kRecBytes + (GK + g) * kChunkScaleBytes);
      const __half2 s0 = as_half2(f2.x & keep[2 * r]), s1 = as_half2(f2.y & keep[2 * r + 1]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t u0 = e < 2 ? w.x : w.x >> 8, u1 = e < 2 ? w.y : w.y >> 8;
        __half2 v0, v1;                                    // 1024 + c, or 1024 + 16 c: to c - 8, then times the scale
        if (e & 1) {
          v0 = __hfma2(as_half2(code_bits(u0, 0x00f000f0u)), sixteenth, bias16);
          v1 = __hfma2(as_half2(code_bits(u1, 0x00f000f0u)), sixteenth, bias16);
        } else {
          v0 = __hadd2(as_half2(code_bits(u0, 0x000f000fu)), bias);
          v1 = __hadd2(as_half2(code_bits(u1, 0x000f000fu)), bias);
        }
        mma16816(st.o[g][e], pa, as_u32(__hmul2(v0, s0)), as_u32(__hmul2(v1, s1)));
      }
    }
  }
}

template <int GK, int GV>
__global__ void __launch_bounds__(kMmThreads, MmaSmem<GK, GV>::kBlocksPerSm) cache4_mma_kernel(const Cache4Args a, int* timeouts) {
  using SM = MmaSmem<GK, GV>;
  constexpr int DV = GV * kGroupDims;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long scratch[kMmWarps + 3];
  __shared__ uint64_t full[kMmWarps][kMmStages];
  __shared__ int stage_base[kMmWarps][kMmStages];
  __shared__ float2 ml[kMmWarps][kMmRows];
  __shared__ int abort_flag;
  volatile int* abort = &abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* ring = smem + warp * kMmStages * SM::kStageBytes;
  float4* sc = reinterpret_cast<float4*>(smem + SM::oC);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMmWarps * kMmStages; ++i) mbar_init(&full[0][0] + i, 1);
    abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }

  Walk<kMmRows, kPageTokens, kMmOver> walk(a);
  int* held = reinterpret_cast<int*>(smem);
  walk.template start<kMmThreads>(scratch, held);
  // once any block has given up on a wait the device's results are void: later blocks skip their work
  if (threadIdx.x == 0) scratch[0] = *(volatile const int*)timeouts != 0 ? 0 : walk.total;
  __syncthreads();
  walk.total = scratch[0];
  __syncthreads();
  long long u = share(walk.total, blockIdx.x, gridDim.x);
  const long long end = share(walk.total, blockIdx.x + 1, gridDim.x);
  SplitRecord out{};
  int place = u < end ? walk.template seek<kMmThreads>(u, scratch, held) : 0;
  fence_proxy_async();          // the requests' units were held where copies go
  __syncthreads();
  int taken = 0;                // half pages this warp has been through: ring place taken % kMmStages, phase of its barrier from the rest
  bool ok = true;
  while (u < end) {
    const Segment& s = walk.s;
    const int p0 = s.lo + place, share_n = (int)min((long long)(walk.length() - place), end - u), n = min(share_n, s.hi - p0);
    if (n <= 0) {               // no more than what ending the segment counts for
      u += share_n;
      place = 0;
      if (u < end) walk.next();
      continue;
    }
    const bool whole = place == 0 && n == s.hi - s.lo;
    const int minpos = s.pos0 + s.row0 / a.hpg, maxpos = s.pos0 + (s.row0 + s.nrows - 1) / a.hpg;
    const int minlow = a.window > 0 ? minpos - a.window + 1 : 0;
    MmaState<GV> st;

    int id = -1, at = 0;        // lane i: page and first key of unit 32 k + i of this piece
    auto look = [&](int k) {
      const int unit = p0 + 32 * k + lane;
      id = -1;
      if (a.n_sel) {
        const int b = lane < a.n_sel ? a.indices[((int64_t)s.tok0 * a.G + s.g) * a.n_sel + lane] : -1;
        const unsigned same = __match_any_sync(0xffffffffu, b);                 // a block named twice counts once
        const int first = b >= 0 && b < a.P && (same & ((1u << lane) - 1u)) == 0 ? b : -1;
        const int mine = __shfl_sync(0xffffffffu, first, unit & 31);
        at = mine * kPageTokens;
        if (unit < p0 + n && mine >= 0) id = a.table[s.r * a.table_ld + mine];
      } else {
        at = unit * kPageTokens;
        if (unit < p0 + n && unit < a.P) id = a.table[s.r * a.table_ld + unit];
      }
      if (id >= a.n_pages) id = -1;
    };
    // warps 0, 1: the halves of even units, 2, 3: of odd ones
    int unit = warp >> 1, filled = taken;
    auto fetch = [&]() {
      while (unit < n) {
        if ((unit >> 1) % 16 == 0 && unit >= 32) look(unit >> 5);
        const int page = __shfl_sync(0xffffffffu, id, unit & 31), key = __shfl_sync(0xffffffffu, at, unit & 31) + (warp & 1) * kMmKeys;
        unit += 2;
        if (page < 0 || key > maxpos || key + kMmKeys <= minlow) continue;
        const int i = filled % kMmStages;
        if (lane == 0) {
          stage_base[warp][i] = key;
          mbar_arrive_expect_tx(&full[warp][i], SM::kStageBytes);
          bulk_load_1d(ring + i * SM::kStageBytes, a.cache + (((int64_t)page * a.G + s.g) * 2 + (warp & 1)) * SM::kStageBytes, SM::kStageBytes, &full[warp][i]);
        }
        ++filled;
        return;
      }
    };
    look(0);
    for (int i = 0; i < kMmStages; ++i) fetch();
    load_rows<GK, GV>(a, s, smem + SM::oQ, sc, st);
    __syncthreads();
    while (taken < filled) {
      const int i = taken % kMmStages;
      ok = mbar_wait_warp(&full[warp][i], (taken / kMmStages) & 1, abort);
      if (!ok) break;
      __syncwarp();
      half_page<GK, GV>(a, s, ring + i * SM::kStageBytes, smem + SM::oQ, sc, stage_base[warp][i], minpos, maxpos, minlow, st);
      ++taken;
      __syncwarp();
      fetch();
    }
    if (!ok && lane == 0)       // let copies in flight land before the block gives its shared memory back
      for (int c = taken; c < filled; ++c) mbar_wait(&full[warp][c % kMmStages], (c / kMmStages) & 1, abort);
    __syncthreads();            // the ring is free: the warps' results take its place
    if (*abort) break;
    float* so = reinterpret_cast<float*>(smem);
    {
      const int r = lane >> 2, j = lane & 3;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float t = st.top[h], sum = st.l[h];
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
          sum += __shfl_xor_sync(0xffffffffu, sum, d);
        }
        // relative to the row's true maximum
        const float f = t == -CUDART_INF_F ? 0.f : ex2((st.m[h] - t) * st.c2[h]);
        if (j == 0) ml[warp][r + 8 * h] = make_float2(t == -CUDART_INF_F ? t : t * st.cl[h], sum * f);
#pragma unroll
        for (int g = 0; g < GV; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<float2*>(so + (warp * kMmRows + r + 8 * h) * DV + g * 32 + e * 8 + 2 * j) =
                make_float2(st.o[g][e][2 * h] * f, st.o[g][e][2 * h + 1] * f);
      }
    }
    __syncthreads();
    float* part = whole ? nullptr : split_part(a, gridDim.x, kMmRows, blockIdx.x, place == 0 ? 1 : 0);
    for (int i = threadIdx.x; i < s.nrows * (DV / 4); i += kMmThreads) {
      const int r = i / (DV / 4), d = i % (DV / 4) * 4;
      float m = -CUDART_INF_F, l = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kMmWarps; ++w) m = fmaxf(m, ml[w][r].x);
#pragma unroll
      for (int w = 0; w < kMmWarps; ++w) {
        const float f = ml[w][r].x == -CUDART_INF_F ? 0.f : ex2((ml[w][r].x - m) * kLog2e);
        const float4 v = *reinterpret_cast<const float4*>(so + (w * kMmRows + r) * DV + d);
        l = fmaf(ml[w][r].y, f, l);
        x.x = fmaf(v.x, f, x.x); x.y = fmaf(v.y, f, x.y); x.z = fmaf(v.z, f, x.z); x.w = fmaf(v.w, f, x.w);
      }
      if (whole) {
        const int64_t row = out_row(a, s, r);
        const float inv = l > 0.f ? 1.f / l : 1.f;
        __nv_bfloat162 b0 = __floats2bfloat162_rn(x.x * inv, x.y * inv), b1 = __floats2bfloat162_rn(x.z * inv, x.w * inv);
        *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + row * DV + d) = make_uint2(*reinterpret_cast<uint32_t*>(&b0), *reinterpret_cast<uint32_t*>(&b1));
        if (d == 0) {
          a.M[row] = m;
          a.L[row] = logf(l);
        }
      } else {
        *reinterpret_cast<float4*>(part + r * DV + d) = x;
        if (d == 0) reinterpret_cast<float2*>(part + kMmRows * DV)[r] = make_float2(m, l);
      }
    }
    if (!whole && place == 0)
      out = SplitRecord{block_of(walk.total, u + s.hi - s.lo - 1, gridDim.x) - (int)blockIdx.x + 1, s.tok0, s.row0, s.nrows, s.g, {}};
    u += share_n;
    place = 0;
    fence_proxy_async();        // the results were written where the next copies go
    __syncthreads();
    if (u < end) walk.next();
  }
  if (threadIdx.x == 0) {
    reinterpret_cast<SplitRecord*>(a.ws)[blockIdx.x] = out;
    if (*abort) report_timeout(timeouts);
  }
  pdl_launch();
}

bool cache4_mma_dims(const Cache4Args& a) {
  return (a.dk == 192 && a.dv == 128) || (a.dk == 128 && a.dv == 128) || (a.dk == 64 && a.dv == 64);
}

template <int GK, int GV>
static int mma_blocks(const Cache4Args& a) { return cache4_grid(a, kMmRows, MmaSmem<GK, GV>::kBlocksPerSm); }

size_t cache4_mma_workspace(const Cache4Args& a) {
  const int blocks = a.dk == 192 ? mma_blocks<6, 4>(a) : a.dk == 128 ? mma_blocks<4, 4>(a) : mma_blocks<2, 2>(a);
  return split_bytes(blocks, kMmRows, a.dv);
}

template <int GK, int GV>
static int launch_mma_t(const Cache4Args& a, int* timeouts, cudaStream_t st) {
  using SM = MmaSmem<GK, GV>;
  auto kern = cache4_mma_kernel<GK, GV>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::kDynamic);
  if (e != cudaSuccess) return fail(NSA_ERR_LAUNCH, "cache4_mma: cannot reserve %d bytes of shared memory: %s", SM::kDynamic, cudaGetErrorString(e));
  const int blocks = mma_blocks<GK, GV>(a);
  {
    KernelTimer kt("cache4_mma", st);
    kern<<<blocks, kMmThreads, SM::kDynamic, st>>>(a, timeouts);
    if (int rc = check_launch("cache4_mma")) return rc;
  }
  return launch_combine(a, blocks, kMmRows, false, st);
}

int launch_mma(const Cache4Args& a, cudaStream_t st) {
  if (timeout_flagged())
    return fail(NSA_ERR_LAUNCH, "cache4_attn: a tensor-core kernel gave up on a barrier wait earlier (device time-out); results since then are "
                "invalid.  nsa_device_timeouts(1) reports and clears the condition");
  int* timeouts = fa_timeout_counter();
  if (!timeouts) return fail(NSA_ERR_LAUNCH, "cache4_mma: cannot set up the time-out record of this device");
  if (a.dk == 192) return launch_mma_t<6, 4>(a, timeouts, st);
  return a.dk == 128 ? launch_mma_t<4, 4>(a, timeouts, st) : launch_mma_t<2, 2>(a, timeouts, st);
}

}  // namespace nsa
