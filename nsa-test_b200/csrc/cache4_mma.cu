// Attention over the 4-bit paged cache for few rows a request (decode, drafted tokens, selected blocks): bf16 queries on mma.m16n8k16 with
// fp16 operands and 32-bit sums.  How the work is cut up: cache4_attn.cuh.
//
// A block of four warps has 16 rows of a kv group and walks the keys a page at a time, brought in by one bulk copy.  A warp forms the logits and
// probabilities of one record (16 keys); through shared memory every warp gets all of them and forms the outputs of 32 value dimensions.
// The cache's layout is the products' B fragment, so a chunk's codes come with one 8-byte load per lane.  (With keys and outputs of its own
// for every warp there was no exchange, but 64 output registers a lane and a loop of 14 KB of instructions: 265 us where this took 249, and
// 28 where this took 24 for the selected blocks of 32 tokens.)
//
// Logits: a nibble c masked out of its word where it lies is the fp16 number c 2^-24 (or 16 c 2^-24: the bits of a number below 2^-13 are its
// multiple of 2^-24), so unpacking costs one AND per two codes; the sums start from -8 sum(q) 2^-24, which turns codes into values.  Each 32
// dimensions are multiplied by their scale in 32 bits.  Queries are scaled to a largest magnitude in [2^14, 2^15) per row (a power of two;
// bf16 has 8 bits, fp16 11, so only elements 2^-20 below the row's largest lose any) and the pairs whose codes arrive 16 times too large are
// divided by 16.  All of it is exact but for the 32-bit sums.
// Outputs: values times scales are exact in fp16; probabilities are rounded to fp16, by 2^-11 (an eighth of the output's own rounding) down to
// 2^-21 of the row's reference, by 2^-32 of the reference below (kProbShift): those of a million keys that all vanish are 2^-12 of the sum.
// The block's reference maximum of a row moves only when a row's maximum outgrows it by 2^8, so what becomes fp16 stays below 2^15.
// What bounds it: no unit is full.  470 instructions per 16 keys of a group (about 280 of them unpack and multiply, the rest is a page's own: masks,
// growth, exchange, fetch) take 45 % of the issue slots and the tensor pipe is active a third of the time; with 16 warps an SM what
// shows is fixed latencies, the two barriers of a page, the math pipes and the fetching of code.  64 requests of up to 32000 tokens: 238 us; without
// unpacking and products the same loop takes 145 (93 % of the copy bandwidth).
#include <algorithm>

#include "attn_args.cuh"
#include "cache4_attn.cuh"
#include "fa_sm100.cuh"
#include "sm100_ptx.cuh"

namespace nsa {

using namespace ptx;

constexpr int kMmThreads = 128, kMmWarps = 4, kMmRows = 16;
constexpr int kMmStages = 3;                         // pages
constexpr int kMmNothing = 0x40000000;               // position of a page that no row sees
constexpr int kMmOver = 1;                           // see Walk
constexpr float kMmGrow = 8.f;                       // log2 units

template <int GK, int GV>
struct MmaSmem {
  static constexpr int kRecBytes = (GK + GV) * kRecBytesPerGroup, kStageBytes = kRecsPerPage * kRecBytes, kRingBytes = kMmStages * kStageBytes;
  static constexpr int oQ = kRingBytes > kHeldBytes ? kRingBytes : kHeldBytes,       // (the requests' units are there at first)
                        oC = oQ + GK * 1024, oP = oC + GK * 128, kDynamic = oP + 2 * 2048;
  static constexpr int kBlocksPerSm = 4;
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
struct MmaState {
  float o[4][4];                               // 32 dimensions of the outputs
  float m[2], lim[2], top[2], l[2], c2[2], cl[2];      // lim: what a maximum has to exceed for m to move; c2: a unit of the sums in log2 logits; cl: 2^24 of them in logits
  int pos[2];
};

// The segment's queries: fragments into shared memory (warp w forms every fourth group's), the rows' constants into registers.
template <int GK>
__device__ __forceinline__ void load_rows(const Cache4Args& a, const Segment& s, uint8_t* sq, float4* sc, MmaState& st) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, j = lane & 3;
  uint4 raw[2][GK];
  float up[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = n + 8 * h, f = s.row0 + i;
    const bool row = i < s.nrows;
    st.pos[h] = row ? s.pos0 + f / a.hpg : -1;
    const __nv_bfloat16* src = (const __nv_bfloat16*)a.q + (s.tok0 + f / a.hpg) * a.sq_tok + (s.g * a.hpg + f % a.hpg) * a.sq_head + 8 * j;
#pragma unroll
    for (int g = 0; g < GK; ++g) raw[h][g] = row ? *reinterpret_cast<const uint4*>(src + g * kGroupDims) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t mx = 0;
#pragma unroll
    for (int g = 0; g < GK; ++g)
      mx = __vmaxu2(__vmaxu2(mx, raw[h][g].x & 0x7fff7fffu), __vmaxu2(__vmaxu2(raw[h][g].y & 0x7fff7fffu, raw[h][g].z & 0x7fff7fffu), raw[h][g].w & 0x7fff7fffu));
    mx = max(mx & 0xffffu, mx >> 16);
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const int k = mx ? min(14 - ((int)(mx >> 7) - 127), 100) : 0;
    // the scale's sign goes into the row, so that a larger sum is always the larger logit; scale 0 is a row of zeros
    up[h] = mx >= 0x7f80 ? CUDART_NAN_F : __uint_as_float((uint32_t)(k + 127) << 23) * (a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : 0.f);
    st.cl[h] = (a.scale == 0.f ? 1.f : fabsf(a.scale)) * __uint_as_float((uint32_t)(127 - k) << 23);
    // Held within 2^100 either way, so that a sum (at most 2^15) times it is finite and -inf times it is -inf: beyond, sums that differ at all
    // are worlds apart or all sums are one.
    st.c2[h] = fminf(fmaxf(st.cl[h] * (16777216.f * kLog2e), 0x1p-100f), 0x1p100f);
    st.m[h] = st.lim[h] = st.top[h] = -CUDART_INF_F;
    st.l[h] = 0.f;
  }
#pragma unroll
  for (int g = 0; g < GK; ++g)
    if ((g & 3) == warp) {
      uint32_t frag[2][4];
      float sum[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t u[4] = {raw[h][g].x, raw[h][g].y, raw[h][g].z, raw[h][g].w};
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = __uint_as_float(u[e] << 16) * up[h];
          x[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u) * up[h];
        }
        sum[h] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {                                 // dimensions e and e + 4: nibbles e, e + 4
          const float w = e & 1 ? 0.0625f : 1.f;
          const __half2 p = __floats2half2_rn(x[e] * w, x[e + 4] * w);
          sum[h] += (__low2float(p) + __high2float(p)) * (e & 1 ? 16.f : 1.f);
          frag[e >> 1][2 * (e & 1) + h] = as_u32(p);
        }
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<uint4*>(sq + (g * 2 + e) * 512 + lane * 16) = make_uint4(frag[e][0], frag[e][1], frag[e][2], frag[e][3]);
      const float c = -4.76837158203125e-07f;                         // -8 * 2^-24
      if (j == 0) sc[g * 8 + n] = make_float4(sum[0] * c, sum[0] * c, sum[1] * c, sum[1] * c);
    }
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) st.o[e][i] = 0.f;
}

// d += a * b for two pairs in one instruction
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%0, %1};\n\t"
      "fma.rn.f32x2 c, a, b, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "+f"(d0), "+f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

template <int GK, int GV>
__global__ void __launch_bounds__(kMmThreads, MmaSmem<GK, GV>::kBlocksPerSm) cache4_mma_kernel(const Cache4Args a, int* timeouts) {
  using SM = MmaSmem<GK, GV>;
  constexpr int DV = GV * kGroupDims, kSplit = 4 / GV;      // warps that share a group of dimensions, each with every kSplit-th record
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long scratch[kMmWarps + 3];
  __shared__ uint64_t full[kMmStages];
  __shared__ int stage_base[kMmStages];
  __shared__ float2 ml[kMmWarps][kMmRows];
  __shared__ int abort_flag;
  volatile int* abort = &abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, j = lane & 3;
  const uint8_t* sq = smem + SM::oQ + lane * 16;
  float4* sc = reinterpret_cast<float4*>(smem + SM::oC);
  uint8_t* sp = smem + SM::oP;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMmStages; ++i) mbar_init(&full[i], 1);
    abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  // once any block has given up on a wait the device's results are void: later blocks skip their work
  const int gave_up = *(volatile const int*)timeouts;

  using W = Walk<kMmRows, kPageTokens, kMmOver, true>;
  __shared__ typename W::Place at_place;
  {
    W walk(a);
    long long* held = reinterpret_cast<long long*>(smem);
    walk.template start<kMmThreads>(scratch, held);
    if (__syncthreads_or(gave_up)) walk.total = 0;
    const long long u = share(walk.total, blockIdx.x, gridDim.x), end = share(walk.total, blockIdx.x + 1, gridDim.x);
    const int place = u < end ? walk.template seek<kMmThreads>(u, scratch, held) : 0;
    if (threadIdx.x == 0) {
      walk.save(at_place, u, end, place);
      reinterpret_cast<SplitRecord*>(a.ws)[blockIdx.x].pieces = 0;
    }
  }
  fence_proxy_async();          // the requests' units were held where copies go
  __syncthreads();
  int i = 0, phase = 0, put = 0;      // ring place of the next page and its barrier's phase, and where the next copy goes
  bool ok = true;
  for (;;) {
    W walk(a);
    long long u, end;
    int place;
    walk.restore(at_place, u, end, place);
    if (u >= end) break;
    const Segment& s = walk.s;
    const int p0 = s.lo + place, share_n = (int)min((long long)(walk.length() - place), end - u), units = min(share_n, s.hi - p0);
    if (units <= 0) {           // no more than what ending the segment counts for
      if (u + share_n < end) walk.next();
      __syncthreads();
      if (threadIdx.x == 0) walk.save(at_place, u + share_n, end, 0);
      __syncthreads();
      continue;
    }
    const int minpos = s.pos0 + s.row0 / a.hpg, maxpos = s.pos0 + (s.row0 + s.nrows - 1) / a.hpg;
    const int minlow = a.window > 0 ? minpos - a.window + 1 : 0;

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
        if (unit < p0 + units && mine >= 0) id = a.table[s.r * a.table_ld + mine];
      } else {
        at = unit * kPageTokens;
        if (unit < p0 + units && unit < a.P) id = a.table[s.r * a.table_ld + unit];
      }
      if (id >= a.n_pages || at > maxpos || at + kPageTokens <= minlow) id = -1;
    };
    // warp 0 brings the pages in; a unit that nothing is seen of takes its turn without a copy
    int unit = 0;
    auto fetch = [&]() {
      if (unit >= units) return;
      if ((unit & 31) == 0) look(unit >> 5);
      const int page = __shfl_sync(0xffffffffu, id, unit & 31), key = __shfl_sync(0xffffffffu, at, unit & 31);
      ++unit;
      if (lane == 0) {
        stage_base[put] = page < 0 ? kMmNothing : key;
        if (page < 0) {
          mbar_arrive(&full[put]);
        } else {
          mbar_arrive_expect_tx(&full[put], SM::kStageBytes);
          bulk_load_1d(smem + put * SM::kStageBytes, a.cache + ((int64_t)page * a.G + s.g) * SM::kStageBytes, SM::kStageBytes, &full[put]);
        }
      }
      if (++put == kMmStages) put = 0;
    };
    if (warp == 0)
      for (int i = 0; i < kMmStages; ++i) fetch();
    MmaState st;
    load_rows<GK>(a, s, smem + SM::oQ, sc, st);
    __syncthreads();
    int done = 0;
    bool far = false;           // some row of this warp has logits beyond kFarLogit
    float bias[2] = {0.f, 0.f}; // of the exponents: kProbShift less the reference
    for (; done < units; ++done) {
      ok = mbar_wait_warp(&full[i], phase, abort);
      // ---- this warp's 16 keys: sums x [tile of 8 keys][row n: keys 2 j, 2 j + 1; row n + 8: the same]
      uint8_t* rec = smem + i * SM::kStageBytes + warp * SM::kRecBytes;
      const int base = stage_base[i] + warp * kRecTokens;
      float x[2][4];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] = 0.f;
#pragma unroll
      for (int g = 0; g < GK; ++g) {
        const uint4 q0 = *reinterpret_cast<const uint4*>(sq + g * 1024), q1 = *reinterpret_cast<const uint4*>(sq + g * 1024 + 512);
        const float4 c0 = sc[g * 8 + n];
        const uint2 w = *reinterpret_cast<const uint2*>(rec + g * kChunkBytes + lane * 8);
        const uint2 f2 = *reinterpret_cast<const uint2*>(rec + (GK + GV) * kChunkBytes + g * kChunkScaleBytes + j * 8);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t b = t ? w.y : w.x, v = b >> 8;
          float c[4];
          mma16816(c, q0, b & 0x000f000fu, b & 0x00f000f0u, c0);
          mma16816(c, q1, v & 0x000f000fu, v & 0x00f000f0u);
          const float2 f = __half22float2(as_half2(t ? f2.y : f2.x));
          fma2(x[t][0], x[t][1], c[0], c[1], f.x, f.y);
          fma2(x[t][2], x[t][3], c[2], c[3], f.x, f.y);
        }
      }
      if (base + kRecTokens - 1 > minpos || (a.window > 0 && base <= maxpos - a.window)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = base + 8 * (e >> 2) + 2 * j + (e & 1), pos = st.pos[e >> 1 & 1];
          if (key > pos || (a.window > 0 && key <= pos - a.window)) x[e >> 2][e & 3] = -CUDART_INF_F;
        }
        // What no row sees may never have been written: nothing of it enters, not as 0 times it either.  Lane t clears the scales of token t.
        if (lane < kRecTokens && (base + lane > maxpos || base + lane < minlow)) {
          uint8_t* to = rec + (GK + GV) * kChunkBytes + GK * kChunkScaleBytes + (4 * (lane >> 1 & 3) + 2 * (lane >> 3) + (lane & 1)) * 2;
#pragma unroll
          for (int g = 0; g < GV; ++g) *reinterpret_cast<uint16_t*>(to + g * kChunkScaleBytes) = 0;
          fence_proxy_async();      // a copy follows these in time
        }
      }
      float mx[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(fmaxf(x[0][2 * h], x[0][2 * h + 1]), fmaxf(x[1][2 * h], x[1][2 * h + 1]));
        st.top[h] = fmaxf(st.top[h], mx[h]);
      }
      // (this barrier also lets go of the page before: every warp has formed its outputs)
      const bool grow = __syncthreads_or(mx[0] > st.lim[0] || mx[1] > st.lim[1] || !ok);
      if (warp == 0 && done > 0) fetch();
      if (grow) {
        if (*abort) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
          if (j == 0) ml[warp][n + 8 * h].x = mx[h];
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = n + 8 * h;
          const float w = fmaxf(fmaxf(ml[0][r].x, ml[1][r].x), fmaxf(ml[2][r].x, ml[3][r].x));
          if (w > st.lim[h]) {
            const float f = ex2((st.m[h] - w) * st.c2[h]);
            st.m[h] = w;
            st.lim[h] = w + kMmGrow / st.c2[h];
            st.l[h] *= f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              st.o[e][2 * h] *= f;
              st.o[e][2 * h + 1] *= f;
            }
          }
        }
        float mc[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) mc[h] = st.m[h] == -CUDART_INF_F ? 0.f : st.m[h] * st.c2[h];
        far = __any_sync(0xffffffffu, fmaxf(fabsf(mc[0]), fabsf(mc[1])) > kFarLogit);
#pragma unroll
        for (int h = 0; h < 2; ++h) bias[h] = far ? kProbShift : kProbShift - mc[h];
      }
      if (far) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] -= st.m[e >> 1 & 1] == -CUDART_INF_F ? 0.f : st.m[e >> 1 & 1];
      }
      uint32_t p[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float e0 = ex2(fmaf(x[t][2 * h], st.c2[h], bias[h])), e1 = ex2(fmaf(x[t][2 * h + 1], st.c2[h], bias[h]));
          st.l[h] += e0 + e1;
          p[t][h] = as_u32(__floats2half2_rn(e0, e1));
        }
      }
      uint8_t* pages_p = sp + (done & 1) * 2048;      // the A fragments of the page's four records
      *reinterpret_cast<uint4*>(pages_p + warp * 512 + lane * 16) = make_uint4(p[0][0], p[0][1], p[1][0], p[1][1]);
      __syncthreads();
      // ---- this warp's 32 dimensions
      const __half2 bias = __float2half2_rn(-1032.f), sixteenth = __float2half2_rn(0.0625f), bias16 = __float2half2_rn(-72.f);
      const uint8_t* values = smem + i * SM::kStageBytes + (GK + warp % GV) * kChunkBytes + lane * 8;
      const uint8_t* vscales = smem + i * SM::kStageBytes + (GK + GV) * kChunkBytes + (GK + warp % GV) * kChunkScaleBytes + j * 8;
#pragma unroll
      for (int k = 0; k < kRecsPerPage / kSplit; ++k) {
        const int r = k * kSplit + warp / GV;
        const uint4 pa = *reinterpret_cast<const uint4*>(pages_p + r * 512 + lane * 16);
        const uint2 w = *reinterpret_cast<const uint2*>(values + r * SM::kRecBytes);
        const uint2 f2 = *reinterpret_cast<const uint2*>(vscales + r * SM::kRecBytes);
        const __half2 s0 = as_half2(f2.x), s1 = as_half2(f2.y);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t b0 = e < 2 ? w.x : w.x >> 8, b1 = e < 2 ? w.y : w.y >> 8;
          __half2 v0, v1;                                    // 1024 + c, or 1024 + 16 c: to c - 8, then times the scale
          if (e & 1) {
            v0 = __hfma2(as_half2(code_bits(b0, 0x00f000f0u)), sixteenth, bias16);
            v1 = __hfma2(as_half2(code_bits(b1, 0x00f000f0u)), sixteenth, bias16);
          } else {
            v0 = __hadd2(as_half2(code_bits(b0, 0x000f000fu)), bias);
            v1 = __hadd2(as_half2(code_bits(b1, 0x000f000fu)), bias);
          }
          mma16816(st.o[e], pa, as_u32(__hmul2(v0, s0)), as_u32(__hmul2(v1, s1)));
        }
      }
      if (++i == kMmStages) {
        i = 0;
        phase ^= 1;
      }
    }
    __syncthreads();
    if (*abort) {               // copies in flight land before the block gives its shared memory back, or another limit ends that (`abort` would at once)
      volatile int overdue = 0;
      for (; threadIdx.x == 0 && done < unit; ++done) {
        mbar_wait(&full[i], phase, &overdue);
        if (++i == kMmStages) {
          i = 0;
          phase ^= 1;
        }
      }
      break;
    }
    // ---- sums over the warps (the walk's place comes back from shared memory: its registers were the loop's)
    walk.restore(at_place, u, end, place);
    const bool whole = place == 0 && units == s.hi - s.lo;
    float f[2], top[2], sum[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = st.top[h];
      sum[h] = st.l[h];
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], d));
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], d);
      }
      if (j == 0) ml[warp][n + 8 * h] = make_float2(top[h], sum[h]);
    }
    float* so = reinterpret_cast<float*>(smem);          // the ring is free
    if (kSplit == 2 && warp >= GV) {
#pragma unroll
      for (int e = 0; e < 16; ++e) so[((warp % GV) * 16 + e) * 32 + lane] = st.o[e >> 2][e & 3];
    }
    __syncthreads();
    float* part = whole ? nullptr : split_part(a, gridDim.x, kMmRows, blockIdx.x, place == 0 ? 1 : 0);
    if (warp < GV) {
      if (kSplit == 2) {
#pragma unroll
        for (int e = 0; e < 16; ++e) st.o[e >> 2][e & 3] += so[(warp * 16 + e) * 32 + lane];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = n + 8 * h;
        if (r >= s.nrows) continue;
        const float2 h0 = ml[0][r], h1 = ml[1][r], h2 = ml[2][r], h3 = ml[3][r];
        sum[h] = (h0.y + h1.y) + (h2.y + h3.y);
        top[h] = max_of_row(fmaxf(fmaxf(h0.x, h1.x), fmaxf(h2.x, h3.x)), sum[h]);
        const float rel = top[h] == -CUDART_INF_F ? 0.f : ex2((st.m[h] - top[h]) * st.c2[h]) * kProbUnshift;       // to the row's true maximum
        const float M = top[h] == -CUDART_INF_F ? top[h] : top[h] * 16777216.f * st.cl[h];
        f[h] = whole ? (sum[h] > 0.f ? 1.f / sum[h] : sum[h]) : rel;
        if (whole) {
          const int64_t row = out_row(a, s, r);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(st.o[e][2 * h] * f[h], st.o[e][2 * h + 1] * f[h]);
            *reinterpret_cast<__nv_bfloat162*>((__nv_bfloat16*)a.out + row * DV + warp * 32 + e * 8 + 2 * j) = b;
          }
          if (warp == 0 && j == 0) {
            a.M[row] = M;
            a.L[row] = logf(sum[h] * rel);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<float2*>(part + r * DV + warp * 32 + e * 8 + 2 * j) = make_float2(st.o[e][2 * h] * f[h], st.o[e][2 * h + 1] * f[h]);
          if (warp == 0 && j == 0) reinterpret_cast<float2*>(part + kMmRows * DV)[r] = make_float2(M, sum[h] * rel);
        }
      }
    }
    if (threadIdx.x == 0 && !whole && place == 0)
      reinterpret_cast<SplitRecord*>(a.ws)[blockIdx.x] =
          SplitRecord{block_of(walk.total, u + s.hi - s.lo - 1, gridDim.x) - (int)blockIdx.x + 1, s.tok0, s.row0, s.nrows, s.g, {}};
    if (u + share_n < end) walk.next();
    fence_proxy_async();        // results were written where the next copies go
    __syncthreads();
    if (threadIdx.x == 0) walk.save(at_place, u + share_n, end, 0);
    __syncthreads();
  }
  if (threadIdx.x == 0 && *abort) report_timeout(timeouts);
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
