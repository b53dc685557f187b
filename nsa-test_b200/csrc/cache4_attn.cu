// Attention of a step's queries over the 4-bit paged cache: see cache4_attn.cuh for how the work is cut up.
#include <algorithm>

#include "attn_args.cuh"
#include "cache4_attn.cuh"
#include "sm100_ptx.cuh"

namespace nsa {

using namespace ptx;

constexpr int kC4Threads = 128, kC4Warps = 4;
constexpr int kC4Stages = 4;                          // records in flight per warp
constexpr int kMasked = 0x40000000;                   // key position that no row sees

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ------------------------------------------------------------------------------------------------
// 32-bit products, any head dims (multiples of 32) and query type: RT rows a tile.  A warp takes a record of 16 keys at a time.
// Logits: lanes 0-15 and 16-31 hold a key each, with the even and the odd groups of dimensions; a lane unpacks 32 dimensions of its key
// and multiplies them into all rows (queries broadcast from shared memory).  Outputs: a lane holds dimensions lane + 32 g.
// ------------------------------------------------------------------------------------------------
template <typename T, int RT, int GV>
struct FmaCore {
  static constexpr int kRows = RT, kBlocksPerSm = 2;
  float o[RT][GV], m[RT], l[RT];
  const float* q;           // shared, [RT][dk], scaled
  float* p;                 // shared, this warp's [RT][16]
  int gk, gv;

  static size_t extra_smem(int dk) { return (size_t)RT * dk * 4 + (size_t)kC4Warps * RT * 16 * 4; }

  __device__ __forceinline__ void begin(const Cache4Args& a, const Segment& s, uint8_t* extra) {
    gk = a.dk / kGroupDims;
    gv = a.dv / kGroupDims;
    float* qs = reinterpret_cast<float*>(extra);
    q = qs;
    p = qs + RT * a.dk + (threadIdx.x >> 5) * RT * 16;
    for (int i = threadIdx.x; i < RT * a.dk; i += kC4Threads) {
      const int r = i / a.dk, d = i - r * a.dk, f = s.row0 + r;
      float x = 0.f;
      if (r < s.nrows) x = Elem<T>::ld((const T*)a.q + (s.tok0 + f / a.hpg) * a.sq_tok + (s.g * a.hpg + f % a.hpg) * a.sq_head + d) * a.scale;
      qs[i] = x;
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      m[r] = -CUDART_INF_F;
      l[r] = 0.f;
#pragma unroll
      for (int g = 0; g < GV; ++g) o[r][g] = 0.f;
    }
    __syncthreads();
  }

  // rows' positions pos0 + (row0 + r) / hpg
  __device__ __forceinline__ void record(const Cache4Args& a, const Segment& s, const uint8_t* rec, int base, int maxpos, int minlow) {
    const int lane = threadIdx.x & 31, dk = a.dk;
    const int key = lane & 15, n = key & 7, t = key >> 3, place = 4 * (n >> 1) + 2 * t + (n & 1);
    const uint8_t* scales = rec + (gk + gv) * kChunkBytes;
    float x[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) x[r] = 0.f;
    for (int g = lane >> 4; g < gk; g += 2) {
      float part[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) part[r] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + g * kChunkBytes + (n * 4 + j) * 8 + t * 4);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)((int)((w >> (4 * e)) & 15u) - 8);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float4 q0 = *reinterpret_cast<const float4*>(q + r * dk + g * 32 + j * 8), q1 = *reinterpret_cast<const float4*>(q + r * dk + g * 32 + j * 8 + 4);
          part[r] = fmaf(q0.x, v[0], fmaf(q0.y, v[1], fmaf(q0.z, v[2], fmaf(q0.w, v[3], part[r]))));
          part[r] = fmaf(q1.x, v[4], fmaf(q1.y, v[5], fmaf(q1.z, v[6], fmaf(q1.w, v[7], part[r]))));
        }
      }
      const float sc = __half2float(reinterpret_cast<const __half*>(scales + g * kChunkScaleBytes)[place]);
#pragma unroll
      for (int r = 0; r < RT; ++r) x[r] = fmaf(part[r], sc, x[r]);
    }
    float f[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      x[r] += __shfl_xor_sync(0xffffffffu, x[r], 16);
      const int pos = r < s.nrows ? s.pos0 + (s.row0 + r) / a.hpg : -1, at = base + key;
      if (at > pos || (a.window > 0 && at <= pos - a.window)) x[r] = -CUDART_INF_F;
      const float mx = fmaxf(m[r], warp_max(x[r]));
      f[r] = m[r] == mx ? 1.f : ex2((m[r] - mx) * kLog2e);
      const float pr = mx == -CUDART_INF_F ? 0.f : ex2((x[r] - mx) * kLog2e);
      m[r] = mx;
      l[r] = l[r] * f[r] + warp_sum(lane < 16 ? pr : 0.f);
      if (lane < 16) p[r * 16 + place] = pr;
    }
    __syncwarp();
#pragma unroll
    for (int g = 0; g < GV; ++g) {
      if (g >= gv) break;
      const uint4* cw = reinterpret_cast<const uint4*>(rec + (gk + g) * kChunkBytes + (lane & 7) * 32);
      const uint4* sw = reinterpret_cast<const uint4*>(scales + (gk + g) * kChunkScaleBytes);
      float v[16];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 c4 = cw[i], s4 = sw[i];
        const uint32_t cu[4] = {c4.x, c4.y, c4.z, c4.w}, su[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int place_ = i * 8 + e, key_ = 8 * (place_ >> 1 & 1) + 2 * (place_ >> 2) + (place_ & 1);
          const uint32_t h = cu[e >> 1] >> (16 * (e & 1) + 4 * (lane >> 3)) & 15u;
          const float sc = __half2float(__ushort_as_half((unsigned short)(su[e >> 1] >> (16 * (e & 1)))));
          // what no row sees may never have been written: nothing of it enters, not as 0 times it either
          v[place_] = base + key_ <= maxpos && base + key_ >= minlow ? (float)((int)h - 8) * sc : 0.f;
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float acc = o[r][g] * f[r];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 pp = *reinterpret_cast<const float4*>(p + r * 16 + 4 * i);
          acc = fmaf(pp.x, v[4 * i], fmaf(pp.y, v[4 * i + 1], fmaf(pp.z, v[4 * i + 2], fmaf(pp.w, v[4 * i + 3], acc))));
        }
        o[r][g] = acc;
      }
    }
    __syncwarp();
  }

  // to shared memory: so [RT][dv], ml [RT]
  __device__ __forceinline__ void finish(const Cache4Args& a, float* so, float2* ml) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
      for (int g = 0; g < GV; ++g)
        if (g < gv) so[r * a.dv + g * 32 + lane] = o[r][g];
      if (lane == 0) ml[r] = make_float2(m[r], l[r]);
    }
  }
};

// ------------------------------------------------------------------------------------------------
// bf16 queries on mma.m16n8k16 with fp16 operands and 32-bit sums, 16 rows a tile, a record of 16 keys at a time per warp.
//
// Logits: a nibble c masked out of its word where it lies is the fp16 number c 2^-24 (or 16 c 2^-24: subnormal numbers are multiples of 2^-24,
// and their bits are the multiple), so unpacking costs one AND per two codes; the sums start from -8 sum(q) 2^-24, which turns codes into
// values.  Each 32 dimensions are multiplied by their scale in 32 bits.  Queries are scaled to a largest magnitude in [2^14, 2^15)
// per row (a power of two; bf16 has 8 bits, fp16 11, so only elements 2^-20 below the row's largest lose any) and the two pairs whose codes
// arrive 16 times too large are divided by 16.  All of it is exact but for the 32-bit sums.
// Outputs: values times scales are exact in fp16; probabilities are rounded to fp16 (2^-11, an eighth of the output's own rounding).
// The reference maximum moves only when a row's maximum outgrows it by a factor of 245, so probabilities stay far below 65504.
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
// (x & mask) | bits in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
  return r;
}

template <int GK, int GV>
struct MmaCore {
  static constexpr int kRows = 16, kBlocksPerSm = GV > 2 ? 3 : 5;
  static constexpr float kGrow = 5.5f;
  uint32_t q[GK][2][4];
  float c0[GK][2];              // -8 sum(q) 2^-24 of rows n, n + 8
  float o[GV][4][4];
  float m[2], top[2], l[2], cl[2];
  int pos[2];

  static size_t extra_smem(int) { return 0; }

  __device__ __forceinline__ void begin(const Cache4Args& a, const Segment& s, uint8_t*) {
    const int lane = threadIdx.x & 31, n = lane >> 2, j = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = n + 8 * h, f = s.row0 + i;
      const bool row = i < s.nrows;
      pos[h] = row ? s.pos0 + f / a.hpg : -1;
      uint4 raw[GK];
      const __nv_bfloat16* src = (const __nv_bfloat16*)a.q + (s.tok0 + f / a.hpg) * a.sq_tok + (s.g * a.hpg + f % a.hpg) * a.sq_head + 8 * j;
      uint32_t mx = 0;
#pragma unroll
      for (int g = 0; g < GK; ++g) {
        raw[g] = row ? *reinterpret_cast<const uint4*>(src + g * kGroupDims) : make_uint4(0, 0, 0, 0);
        const uint32_t u[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = max(mx, max(u[e] & 0x7fffu, u[e] >> 16 & 0x7fffu));
      }
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const int k = mx ? min(14 - ((int)(mx >> 7) - 127), 100) : 0;
      const float up = __uint_as_float((uint32_t)(min(k, 100) + 127) << 23);
      cl[h] = a.scale * __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
      for (int g = 0; g < GK; ++g) {
        const uint32_t u[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
        float x[8], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = __uint_as_float(u[e] << 16) * up;
          x[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u) * up;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {                                 // dimensions e and e + 4: nibbles e, e + 4
          const float w = e & 1 ? 0.0625f : 1.f;
          const __half2 p = __floats2half2_rn(x[e] * w, x[e + 4] * w);
          sum += (__low2float(p) + __high2float(p)) * (e & 1 ? 16.f : 1.f);
          q[g][e >> 1][2 * (e & 1) + h] = as_u32(p);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        c0[g][h] = sum * -4.76837158203125e-07f;                      // 8 * 2^-24
      }
      m[h] = top[h] = -CUDART_INF_F;
      l[h] = 0.f;
    }
#pragma unroll
    for (int g = 0; g < GV; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[g][e][i] = 0.f;
  }

  __device__ __forceinline__ void record(const Cache4Args& a, const Segment& s, const uint8_t* rec, int base, int maxpos, int minlow) {
    const int lane = threadIdx.x & 31, j = lane & 3;
    const uint8_t* scales = rec + (GK + GV) * kChunkBytes + j * 8;
    float x[2][4];                  // [tile of 8 keys][row n: keys 2 j, 2 j + 1; row n + 8: the same]
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i >> 2][i & 3] = 0.f;
#pragma unroll
    for (int g = 0; g < GK; ++g) {
      const uint2 w = *reinterpret_cast<const uint2*>(rec + g * kChunkBytes + lane * 8);
      const uint2 sc = *reinterpret_cast<const uint2*>(scales + g * kChunkScaleBytes);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t u = t ? w.y : w.x, v = u >> 8;
        float c[4] = {c0[g][0], c0[g][0], c0[g][1], c0[g][1]};
        mma16816(c, q[g][0], u & 0x000f000fu, u & 0x00f000f0u);
        mma16816(c, q[g][1], v & 0x000f000fu, v & 0x00f000f0u);
        const float2 f = __half22float2(as_half2(t ? sc.y : sc.x));
        x[t][0] = fmaf(c[0], f.x, x[t][0]);
        x[t][1] = fmaf(c[1], f.y, x[t][1]);
        x[t][2] = fmaf(c[2], f.x, x[t][2]);
        x[t][3] = fmaf(c[3], f.y, x[t][3]);
      }
    }
    const bool partial = base + kRecTokens - 1 > s.pos0 + s.row0 / a.hpg || (a.window > 0 && base <= maxpos - a.window);
    float mx[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[t][i] = x[t][i] * 16777216.f * cl[i >> 1];
        if (partial) {
          const int at = base + 8 * t + 2 * j + (i & 1), p = pos[i >> 1];
          if (at > p || (a.window > 0 && at <= p - a.window)) x[t][i] = -CUDART_INF_F;
        }
        mx[i >> 1] = fmaxf(mx[i >> 1], x[t][i]);
      }
    top[0] = fmaxf(top[0], mx[0]);
    top[1] = fmaxf(top[1], mx[1]);
    if (__any_sync(0xffffffffu, mx[0] > m[0] + kGrow || mx[1] > m[1] + kGrow)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float w = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 2));
        if (w > m[h] + kGrow) {
          const float f = ex2((m[h] - w) * kLog2e);
          m[h] = w;
          l[h] *= f;
#pragma unroll
          for (int g = 0; g < GV; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[g][e][2 * h] *= f;
              o[g][e][2 * h + 1] *= f;
            }
        }
      }
    }
    const float b0 = m[0] == -CUDART_INF_F ? 0.f : m[0] * -kLog2e, b1 = m[1] == -CUDART_INF_F ? 0.f : m[1] * -kLog2e;
    uint32_t p[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float p0 = ex2(fmaf(x[t][0], kLog2e, b0)), p1 = ex2(fmaf(x[t][1], kLog2e, b0));
      const float p2 = ex2(fmaf(x[t][2], kLog2e, b1)), p3 = ex2(fmaf(x[t][3], kLog2e, b1));
      l[0] += p0 + p1;
      l[1] += p2 + p3;
      p[2 * t] = as_u32(__floats2half2_rn(p0, p1));
      p[2 * t + 1] = as_u32(__floats2half2_rn(p2, p3));
    }
    // what no row sees may never have been written: nothing of it enters, not as 0 times it either
    uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
    if (base + kRecTokens - 1 > maxpos || base < minlow) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int at = base + 8 * t + 2 * j;
        keep[t] = (at <= maxpos && at >= minlow ? 0xffffu : 0u) | (at + 1 <= maxpos && at + 1 >= minlow ? 0xffff0000u : 0u);
      }
    }
    const __half2 bias = __float2half2_rn(-1032.f), sixteenth = __float2half2_rn(0.0625f), bias16 = __float2half2_rn(-72.f);
#pragma unroll
    for (int g = 0; g < GV; ++g) {
      const uint2 w = *reinterpret_cast<const uint2*>(rec + (GK + g) * kChunkBytes + lane * 8);
      const uint2 sc = *reinterpret_cast<const uint2*>(scales + (GK + g) * kChunkScaleBytes);
      const __half2 s0 = as_half2(sc.x & keep[0]), s1 = as_half2(sc.y & keep[1]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t u0 = e < 2 ? w.x : w.x >> 8, u1 = e < 2 ? w.y : w.y >> 8;
        __half2 v0, v1;                                    // 1024 + c, or 1024 + 16 c: to c - 8, then times the scale
        if (e & 1) {
          v0 = __hfma2(as_half2(and_or(u0, 0x00f000f0u, 0x64006400u)), sixteenth, bias16);
          v1 = __hfma2(as_half2(and_or(u1, 0x00f000f0u, 0x64006400u)), sixteenth, bias16);
        } else {
          v0 = __hadd2(as_half2(and_or(u0, 0x000f000fu, 0x64006400u)), bias);
          v1 = __hadd2(as_half2(and_or(u1, 0x000f000fu, 0x64006400u)), bias);
        }
        mma16816(o[g][e], p, as_u32(__hmul2(v0, s0)), as_u32(__hmul2(v1, s1)));
      }
    }
  }

  __device__ __forceinline__ void finish(const Cache4Args& a, float* so, float2* ml) {
    const int lane = threadIdx.x & 31, n = lane >> 2, j = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float t = top[h], sum = l[h];
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
      }
      // results relative to the row's true maximum
      const float f = t == -CUDART_INF_F ? 0.f : ex2((m[h] - t) * kLog2e);
      if (j == 0) ml[n + 8 * h] = make_float2(t, sum * f);
#pragma unroll
      for (int g = 0; g < GV; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<float2*>(so + (n + 8 * h) * (GV * 32) + g * 32 + e * 8 + 2 * j) = make_float2(o[g][e][2 * h] * f, o[g][e][2 * h + 1] * f);
    }
  }
};

// ------------------------------------------------------------------------------------------------
template <typename T, class Core>
__global__ void __launch_bounds__(kC4Threads, Core::kBlocksPerSm) cache4_attn_kernel(const Cache4Args a) {
  constexpr int ROWS = Core::kRows;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ long long scratch[kC4Warps + 3];
  __shared__ int stage_base[kC4Warps][kC4Stages];
  __shared__ float2 ml[kC4Warps][ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int groups = (a.dk + a.dv) / kGroupDims, rec_bytes = groups * kRecBytesPerGroup;
  uint8_t* ring = smem + warp * kC4Stages * rec_bytes;
  uint8_t* extra = smem + kC4Warps * kC4Stages * rec_bytes;

  Walk<ROWS> walk(a);
  walk.template start<kC4Threads>(scratch);
  long long u = share(walk.total, blockIdx.x, gridDim.x);
  const long long end = share(walk.total, blockIdx.x + 1, gridDim.x);
  SplitRecord out{};
  int place = u < end ? walk.template seek<kC4Threads>(u, scratch) : 0;
  while (u < end) {
    const Segment& s = walk.s;
    const int p0 = s.lo + place, n = (int)min((long long)(s.hi - p0), end - u);
    const bool whole = place == 0 && n == s.hi - s.lo;
    const int maxpos = s.pos0 + (s.row0 + s.nrows - 1) / a.hpg;
    const int minlow = a.window > 0 ? s.pos0 + s.row0 / a.hpg - a.window + 1 : 0;
    Core core;
    core.begin(a, s, extra);

    int id = -1, at = 0;       // lane i: page and first key of unit 32 k + i of this piece
    auto fetch = [&](int i) {
      if (i < n && (i & 31) == 0) {
        id = -1;
        const int unit = p0 + i + lane;
        if (a.n_sel) {
          const int b = lane < a.n_sel ? a.indices[((int64_t)s.tok0 * a.G + s.g) * a.n_sel + lane] : -1;
          const unsigned same = __match_any_sync(0xffffffffu, b);                 // a block named twice counts once
          const int first = b >= 0 && b < a.P && (same & ((1u << lane) - 1u)) == 0 ? b : -1;
          const int mine = __shfl_sync(0xffffffffu, first, unit & 31);
          at = mine * kPageTokens;
          if (unit < s.hi && mine >= 0) id = a.table[s.r * a.table_ld + mine];
        } else {
          at = unit * kPageTokens;
          if (unit < s.hi && unit < a.P) id = a.table[s.r * a.table_ld + unit];
        }
        if (id >= a.n_pages) id = -1;
      }
      if (i < n) {
        const int page = __shfl_sync(0xffffffffu, id, i & 31), key = __shfl_sync(0xffffffffu, at, i & 31) + warp * kRecTokens;
        const bool use = page >= 0 && key <= maxpos && key + kRecTokens > minlow;
        if (use) {
          const uint8_t* src = a.cache + (((int64_t)page * a.G + s.g) * kRecsPerPage + warp) * rec_bytes;
          uint8_t* dst = ring + (i % kC4Stages) * rec_bytes;
          for (int c = lane * 16; c < rec_bytes; c += 512) cp_async16(dst + c, src + c);
        }
        if (lane == 0) stage_base[warp][i % kC4Stages] = use ? key : kMasked;
      }
      cp_commit();
    };
    for (int i = 0; i < kC4Stages - 1; ++i) fetch(i);
    for (int i = 0; i < n; ++i) {
      fetch(i + kC4Stages - 1);
      cp_wait<kC4Stages - 1>();
      __syncwarp();
      const int base = stage_base[warp][i % kC4Stages];
      if (base != kMasked) core.record(a, s, ring + (i % kC4Stages) * rec_bytes, base, maxpos, minlow);
      __syncwarp();
    }
    cp_wait<0>();
    __syncthreads();            // the ring is free: the warps' results take its place
    float* so = reinterpret_cast<float*>(smem);
    core.finish(a, so + warp * ROWS * a.dv, ml[warp]);
    __syncthreads();
    float* part = whole ? nullptr : split_part(a, gridDim.x, ROWS, blockIdx.x, place == 0 ? 1 : 0);
    for (int i = threadIdx.x; i < s.nrows * a.dv; i += kC4Threads) {
      const int r = i / a.dv, d = i - r * a.dv;
      float m = -CUDART_INF_F, l = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < kC4Warps; ++w) m = fmaxf(m, ml[w][r].x);
#pragma unroll
      for (int w = 0; w < kC4Warps; ++w) {
        const float f = ml[w][r].x == -CUDART_INF_F ? 0.f : ex2((ml[w][r].x - m) * kLog2e);
        l = fmaf(ml[w][r].y, f, l);
        x = fmaf(so[(w * ROWS + r) * a.dv + d], f, x);
      }
      if (whole) {
        const int64_t row = out_row(a, s, r);
        Elem<T>::st((T*)a.out + row * a.dv + d, l > 0.f ? x / l : x);
        if (d == 0) {
          a.M[row] = m;
          a.L[row] = logf(l);
        }
      } else {
        part[i] = x;
        if (d == 0) reinterpret_cast<float2*>(part + ROWS * a.dv)[r] = make_float2(m, l);
      }
    }
    if (!whole && place == 0) out = SplitRecord{1, s.tok0, s.row0, s.nrows, s.g, 0, u, u + s.hi - s.lo, walk.total};
    u += n;
    place = 0;
    __syncthreads();
    if (u < end) walk.next();
  }
  if (threadIdx.x == 0) reinterpret_cast<SplitRecord*>(a.ws)[blockIdx.x] = out;
}

// Joins the partial results of the rows of one split segment: block (owner, first row).  The pieces are the owner's last segment and the
// first segments of the blocks after it; four warps take every fourth of them, in a fixed order.
constexpr int kCombineRows = 32;           // rows of an owner at once
template <typename T>
__global__ void __launch_bounds__(128) cache4_combine_kernel(const Cache4Args a, int blocks, int rows) {
  const SplitRecord rec = reinterpret_cast<const SplitRecord*>(a.ws)[blockIdx.x];
  if (!rec.open || (int)blockIdx.y >= rec.nrows) return;
  __shared__ float acc[4][kMaxHeadDim];
  __shared__ float2 ml[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int last = blockIdx.x;                   // the last block that has a unit of the segment
  for (int up = blocks; up - last > 1;) {
    const int mid = (last + up) >> 1;
    if (share(rec.total, mid, blocks) < rec.last) last = mid; else up = mid;
  }
  for (int r = blockIdx.y; r < rec.nrows; r += kCombineRows) {
    float m = -CUDART_INF_F, l = 0.f, x[kMaxHeadDim / 32] = {};
    for (int c = blockIdx.x + warp; c <= last; c += 4) {
      if (c > (int)blockIdx.x && share(rec.total, c, blocks) == share(rec.total, c + 1, blocks)) continue;   // more blocks than units
      const float* part = split_part(a, blocks, rows, c, c == (int)blockIdx.x ? 1 : 0);
      const float2 h = reinterpret_cast<const float2*>(part + rows * a.dv)[r];
      if (h.x == -CUDART_INF_F) continue;
      const float mx = fmaxf(m, h.x), f0 = m == -CUDART_INF_F ? 0.f : ex2((m - mx) * kLog2e), f1 = ex2((h.x - mx) * kLog2e);
      m = mx;
      l = l * f0 + h.y * f1;
#pragma unroll
      for (int g = 0; g < kMaxHeadDim / 32; ++g)
        if (g * 32 < a.dv) x[g] = x[g] * f0 + part[r * a.dv + g * 32 + lane] * f1;
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < kMaxHeadDim / 32; ++g)
      if (g * 32 < a.dv) acc[warp][g * 32 + lane] = x[g];
    if (lane == 0) ml[warp] = make_float2(m, l);
    __syncthreads();
    float M = -CUDART_INF_F, sum = 0.f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, ml[w].x);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = ml[w].x == -CUDART_INF_F ? 0.f : ex2((ml[w].x - M) * kLog2e);
      sum = fmaf(ml[w].y, f[w], sum);
    }
    Segment s;
    s.tok0 = rec.tok0; s.row0 = rec.row0; s.g = rec.g;
    const int64_t row = out_row(a, s, r);
    for (int d = threadIdx.x; d < a.dv; d += 128) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) v = fmaf(acc[w][d], f[w], v);
      Elem<T>::st((T*)a.out + row * a.dv + d, sum > 0.f ? v / sum : v);
    }
    if (threadIdx.x == 0) {
      a.M[row] = M;
      a.L[row] = logf(sum);
    }
  }
}

int launch_combine(const Cache4Args& a, int blocks, int rows, bool f32, cudaStream_t st) {
  KernelTimer kt("cache4_combine", st);
  const dim3 grid(blocks, std::min(rows, kCombineRows));
  if (f32) cache4_combine_kernel<float><<<grid, 128, 0, st>>>(a, blocks, rows);
  else cache4_combine_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(a, blocks, rows);
  return check_launch("cache4_combine");
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int kFmaRows = 8;
constexpr int kC4Smem = 227 * 1024 - 4096;

// rows (new tokens times heads of a group) from which a request goes to the tensor-memory kernel
constexpr int kChunkRows = 128;

static size_t ring_bytes(int dk, int dv) { return (size_t)kC4Warps * kC4Stages * ((dk + dv) / kGroupDims) * kRecBytesPerGroup; }

// thread blocks of a launch: what the device holds at once, or as many as there can be units
static int grid_blocks(const Cache4Args& a, int rows, int per_sm) {
  const long long tiles = a.n_sel ? (long long)a.N * ((a.hpg + rows - 1) / rows) : ((long long)a.N * a.hpg + rows - 1) / rows + a.S;
  const long long units = tiles * a.G * (a.n_sel ? a.n_sel : std::max(a.P, 1));
  return (int)std::min<long long>(per_sm * 148, std::max<long long>(units, 1));
}

template <typename T, class Core>
static size_t core_workspace(const Cache4Args& a) {
  return split_bytes(grid_blocks(a, Core::kRows, Core::kBlocksPerSm), Core::kRows, a.dv);
}
template <typename T, class Core>
static int launch_core(const Cache4Args& a, const char* name, cudaStream_t st) {
  auto kern = cache4_attn_kernel<T, Core>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kC4Smem);
  if (e != cudaSuccess) return fail(NSA_ERR_LAUNCH, "cache4_attn: cannot reserve shared memory: %s", cudaGetErrorString(e));
  const int blocks = grid_blocks(a, Core::kRows, Core::kBlocksPerSm);
  {
    KernelTimer kt(name, st);
    kern<<<blocks, kC4Threads, ring_bytes(a.dk, a.dv) + Core::extra_smem(a.dk), st>>>(a);
    if (int rc = check_launch("cache4_attn")) return rc;
  }
  return launch_combine(a, blocks, Core::kRows, sizeof(T) == 4, st);
}

// The tensor-core kernel takes bf16 queries of the head dims that the other tensor-core kernels know; its rows are loaded 16 bytes at a time.
static bool mma_dims(const Cache4Args& a, int dtype) {
  return dtype == NSA_BF16 && ((a.dk == 192 && a.dv == 128) || (a.dk == 128 && a.dv == 128) || (a.dk == 64 && a.dv == 64));
}
static bool mma_aligned(const Cache4Args& a) { return (uintptr_t)a.q % 16 == 0 && a.sq_tok % 8 == 0 && a.sq_head % 8 == 0; }

#define NSA_C4_FMA(FN, ...)                                                                              \
  (dtype == NSA_F32 ? (a.dv > 128 ? FN<float, FmaCore<float, kFmaRows, 8>>(__VA_ARGS__)                  \
                                  : FN<float, FmaCore<float, kFmaRows, 4>>(__VA_ARGS__))                 \
                    : (a.dv > 128 ? FN<__nv_bfloat16, FmaCore<__nv_bfloat16, kFmaRows, 8>>(__VA_ARGS__)  \
                                  : FN<__nv_bfloat16, FmaCore<__nv_bfloat16, kFmaRows, 4>>(__VA_ARGS__)))
#define NSA_C4_MMA(FN, ...)                                                   \
  (a.dk == 192   ? FN<__nv_bfloat16, MmaCore<6, 4>>(__VA_ARGS__)              \
   : a.dk == 128 ? FN<__nv_bfloat16, MmaCore<4, 4>>(__VA_ARGS__)              \
                 : FN<__nv_bfloat16, MmaCore<2, 2>>(__VA_ARGS__))

static int cache4_args(const nsa_cache4_desc* d, Cache4Args& a) {
  NSA_REQUIRE(d, "cache4_attn: null descriptor");
  NSA_REQUIRE(d->N >= 0 && d->S >= 0 && d->P >= 0 && d->n_pages >= 0, "cache4_attn: bad sizes %d/%d/%d/%d", d->N, d->S, d->P, d->n_pages);
  NSA_REQUIRE(d->H > 0 && d->G > 0 && d->H % d->G == 0 && d->H <= 65535, "cache4_attn: bad H/G = %d/%d", d->H, d->G);
  NSA_REQUIRE(d->dk > 0 && d->dv > 0 && d->dk <= kMaxHeadDim && d->dv <= kMaxHeadDim && d->dk % kGroupDims == 0 && d->dv % kGroupDims == 0,
              "cache4_attn: head dims %d/%d are no multiples of %d up to %d", d->dk, d->dv, kGroupDims, kMaxHeadDim);
  NSA_REQUIRE(d->dtype == NSA_F32 || d->dtype == NSA_BF16, "cache4_attn: unsupported dtype %d", d->dtype);
  NSA_REQUIRE(d->n_sel >= 0 && d->n_sel <= kSelMax, "cache4_attn: %d selected blocks, at most %d", d->n_sel, kSelMax);
  NSA_REQUIRE(d->window >= 0 && (d->window == 0 || d->n_sel == 0), "cache4_attn: a window and selected blocks do not go together");
  NSA_REQUIRE(d->max_new >= 0, "cache4_attn: negative max_new");
  NSA_REQUIRE(d->P <= 1 << 23, "cache4_attn: %d pages a request, at most %d", d->P, 1 << 23);
  NSA_REQUIRE((int64_t)d->N * d->H <= 0x7fffffffll / 4, "cache4_attn: %d tokens of %d heads in one call", d->N, d->H);
  a.q = d->q; a.cache = (const uint8_t*)d->cache; a.table = d->table; a.lengths = d->lengths; a.starts = d->starts;
  a.indices = d->indices; a.out = d->out; a.L = d->L; a.M = d->M;
  a.sq_tok = d->sq[0]; a.sq_head = d->sq[1]; a.table_ld = d->table_ld;
  a.N = d->N; a.S = d->S; a.P = d->P; a.H = d->H; a.G = d->G; a.hpg = d->H / d->G; a.dk = d->dk; a.dv = d->dv;
  a.n_pages = d->n_pages; a.n_sel = d->n_sel; a.window = std::min(d->window, 1 << 30); a.scale = d->scale;
  a.rows_lo = 0; a.rows_hi = 0x7fffffff; a.ws = nullptr;
  return NSA_OK;
}

}  // namespace nsa

using namespace nsa;

extern "C" NSA_API size_t nsa_cache4_attn_workspace_bytes(const nsa_cache4_desc* desc) {
  Cache4Args a;
  if (cache4_args(desc, a) != NSA_OK || a.N == 0 || a.S == 0) return 0;
  const int dtype = desc->dtype;
  const size_t fma = NSA_C4_FMA(core_workspace, a);
  if (!mma_dims(a, dtype)) return fma;
  const size_t mma = NSA_C4_MMA(core_workspace, a);
  return std::max({fma, mma, a.n_sel ? 0 : cache4_chunk_workspace(a)});
}

extern "C" NSA_API int nsa_cache4_attn_fwd(const nsa_cache4_desc* desc, void* workspace, size_t workspace_bytes, void* stream) {
  Cache4Args a;
  if (int rc = cache4_args(desc, a)) return rc;
  if (a.N == 0 || a.S == 0) return NSA_OK;
  NSA_REQUIRE(a.q && a.starts && a.lengths && a.out && a.L && a.M && (a.P == 0 || (a.table && a.table_ld >= a.P)) && (a.n_pages == 0 || a.cache) &&
                  (a.n_sel == 0 || a.indices), "cache4_attn: null pointer");
  NSA_REQUIRE((uintptr_t)a.cache % 16 == 0, "cache4_attn: the cache must be 16-byte aligned");
  const size_t need = nsa_cache4_attn_workspace_bytes(desc);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
    return fail(NSA_ERR_WORKSPACE, "cache4_attn: needs %zu bytes of 16-byte aligned scratch, got %zu", need, workspace_bytes);
  a.ws = (uint8_t*)workspace;
  cudaStream_t st = (cudaStream_t)stream;
  const int dtype = desc->dtype;
  if (mma_dims(a, dtype) && mma_aligned(a)) {
    // Each request goes to the kernel that suits its rows, by their numbers on the device; a launch that the host can tell to be empty is left out.
    const int most = desc->max_new > 0 ? std::min(desc->max_new, a.N) : a.N;
    const bool chunks = a.n_sel == 0 && (int64_t)most * a.hpg >= kChunkRows;
    const bool uniform = desc->max_new > 0 && (int64_t)a.S * desc->max_new == a.N && chunks;
    if (chunks) {
      a.rows_lo = kChunkRows;
      if (int rc = launch_chunk(a, st)) return rc;
      a.rows_lo = 0;
      a.rows_hi = kChunkRows;
    }
    return uniform ? NSA_OK : NSA_C4_MMA(launch_core, a, "cache4_attn_mma", st);
  }
  return NSA_C4_FMA(launch_core, a, "cache4_attn_fma", st);
}
