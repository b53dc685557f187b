// Attention of a step's queries over the 4-bit paged cache: see cache4_attn.cuh for how the work is cut up.
#include <algorithm>
#include <cmath>

#include "attn_args.cuh"
#include "cache4_attn.cuh"
#include "fa_sm100.cuh"
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
      if (r < s.nrows) x = Elem<T>::ld((const T*)a.q + (s.tok0 + f / a.hpg) * a.sq_tok + (s.g * a.hpg + f % a.hpg) * a.sq_head + d);
      x = isfinite(x) ? x * a.scale : CUDART_NAN_F;
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
      const float pr = x[r] == -CUDART_INF_F ? 0.f : ex2((x[r] - mx) * kLog2e);
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
  uint8_t* extra = smem + max(kC4Warps * kC4Stages * rec_bytes, kHeldBytes);

  Walk<ROWS, kPageTokens, 1, true> walk(a);
  long long* held = reinterpret_cast<long long*>(smem);
  walk.template start<kC4Threads>(scratch, held);
  long long u = share(walk.total, blockIdx.x, gridDim.x);
  const long long end = share(walk.total, blockIdx.x + 1, gridDim.x);
  SplitRecord out{};
  int place = u < end ? walk.template seek<kC4Threads>(u, scratch, held) : 0;
  __syncthreads();
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
          a.M[row] = max_of_row(m, l);
          a.L[row] = logf(l);
        }
      } else {
        part[i] = x;
        if (d == 0) reinterpret_cast<float2*>(part + ROWS * a.dv)[r] = make_float2(max_of_row(m, l), l);
      }
    }
    if (!whole && place == 0)
      out = SplitRecord{block_of(walk.total, u + s.hi - s.lo - 1, gridDim.x) - (int)blockIdx.x + 1, s.tok0, s.row0, s.nrows, s.g, {}};
    u += share_n;
    place = 0;
    __syncthreads();
    if (u < end) walk.next();
  }
  if (threadIdx.x == 0) reinterpret_cast<SplitRecord*>(a.ws)[blockIdx.x] = out;
  pdl_launch();
}

// Joins the partial results of a split segment's rows.  The pieces are the owner's last segment and the first segments of the blocks
// after it.  WARPS = 4: a block has one row and its warps share the pieces (few rows, possibly hundreds of pieces); 1: a warp has a row
// (the many rows of a chunk, whose segments fall into two or three pieces).  Weights first, 32 pieces at a time with a lane each, then the
// weighted sum, whose loads do not depend on one another; the order is fixed.
template <typename T, int WARPS>
__global__ void __launch_bounds__(128) cache4_combine_kernel(const Cache4Args a, int blocks, int rows) {
  pdl_wait();
  const SplitRecord rec = reinterpret_cast<const SplitRecord*>(a.ws)[blockIdx.x];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = WARPS == 4 ? blockIdx.y : blockIdx.y * 4 + warp;
  if (rec.pieces == 0 || (WARPS == 4 ? (int)blockIdx.y : (int)blockIdx.y * 4) >= rec.nrows) return;
  if (WARPS == 1 && r >= rec.nrows) return;
  __shared__ float acc[WARPS == 4 ? 4 : 1][kMaxHeadDim];
  __shared__ float2 ml[4];
  const int q0 = WARPS == 4 ? warp : 0;                   // this warp's pieces: q0, q0 + WARPS, ...
  const float* first = split_part(a, blocks, rows, blockIdx.x, 1);
  const float* others = split_part(a, blocks, rows, blockIdx.x, 0);
  const size_t step = 2 * split_part_floats(rows, a.dv);
  auto part = [&](int p) { return p == 0 ? first : others + (size_t)p * step; };
  float m = -CUDART_INF_F, l = 0.f;
  float4 x[2] = {};                                       // dimensions 4 lane + 128 i
  for (int p0 = q0; p0 < rec.pieces; p0 += 32 * WARPS) {
    const int p = p0 + lane * WARPS;
    float2 h = make_float2(-CUDART_INF_F, 0.f);
    if (p < rec.pieces) h = reinterpret_cast<const float2*>(part(p) + rows * a.dv)[r];
    const float mx = fmaxf(m, warp_max(h.x));
    if (mx == -CUDART_INF_F && !__any_sync(0xffffffffu, h.x != h.x)) continue;      // (a row that is NaN goes on, whatever the maximum)
    const float f = ex2((m - mx) * kLog2e), w = ex2((h.x - mx) * kLog2e);
    m = mx;
    l = l * f + warp_sum(h.y * w);
#pragma unroll
    for (int i = 0; i < 2; ++i) { x[i].x *= f; x[i].y *= f; x[i].z *= f; x[i].w *= f; }
    const int n = min(32, (rec.pieces - p0 + WARPS - 1) / WARPS);
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      const float4* src = reinterpret_cast<const float4*>(part(p0 + k * WARPS) + r * a.dv);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (lane * 4 + i * 128 < a.dv) {
          const float4 v = src[lane + i * 32];
          x[i].x = fmaf(v.x, wk, x[i].x); x[i].y = fmaf(v.y, wk, x[i].y); x[i].z = fmaf(v.z, wk, x[i].z); x[i].w = fmaf(v.w, wk, x[i].w);
        }
    }
  }
  Segment s;
  s.tok0 = rec.tok0; s.row0 = rec.row0; s.g = rec.g;
  const int64_t row = out_row(a, s, r);
  float f[4] = {1.f, 0.f, 0.f, 0.f};
  if (WARPS == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (lane * 4 + i * 128 < a.dv) *reinterpret_cast<float4*>(&acc[warp][lane * 4 + i * 128]) = x[i];
    if (lane == 0) ml[warp] = make_float2(m, l);
    __syncthreads();
    if (warp > 0) return;
    m = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
    l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = ml[w].x == -CUDART_INF_F ? 0.f : ex2((ml[w].x - m) * kLog2e);
      l = fmaf(ml[w].y, f[w], l);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (lane * 4 + i * 128 < a.dv) {
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(&acc[w][lane * 4 + i * 128]);
          x[i].x = fmaf(v.x, f[w], x[i].x); x[i].y = fmaf(v.y, f[w], x[i].y); x[i].z = fmaf(v.z, f[w], x[i].z); x[i].w = fmaf(v.w, f[w], x[i].w);
        }
      }
  }
  const float inv = l > 0.f ? 1.f / l : 1.f;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane * 4 + i * 128 < a.dv) {
      T* to = (T*)a.out + row * a.dv + lane * 4 + i * 128;
      Elem<T>::st(to, x[i].x * inv); Elem<T>::st(to + 1, x[i].y * inv); Elem<T>::st(to + 2, x[i].z * inv); Elem<T>::st(to + 3, x[i].w * inv);
    }
  if (lane == 0) {
    a.M[row] = max_of_row(m, l);
    a.L[row] = logf(l);
  }
}

// The launch overlaps the end of the kernel before it (programmatic dependent launch).
int launch_combine(const Cache4Args& a, int blocks, int rows, bool f32, cudaStream_t st) {
  KernelTimer kt("cache4_combine", st);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, rows > 16 ? (rows + 3) / 4 : rows);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = f32         ? cudaLaunchKernelEx(&cfg, cache4_combine_kernel<float, 4>, a, blocks, rows)
                        : rows > 16 ? cudaLaunchKernelEx(&cfg, cache4_combine_kernel<__nv_bfloat16, 1>, a, blocks, rows)
                                    : cudaLaunchKernelEx(&cfg, cache4_combine_kernel<__nv_bfloat16, 4>, a, blocks, rows);
  if (e != cudaSuccess) return fail(NSA_ERR_LAUNCH, "cache4_combine: %s", cudaGetErrorString(e));
  return NSA_OK;
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int kFmaRows = 8;
constexpr int kC4Smem = 227 * 1024 - 4096;

// Rows (new tokens times heads of a group) from which a request goes to the tensor-memory kernel: it does 256 rows for the price of one,
// the mma.sync kernel 16 at a time.  us, it against the mma.sync kernel:
//   16 requests of up to 8000 tokens, 48 / 64 / 80 / 96 rows   192/128: 70:63 71:80 71:98 72:114   128/128: 41:36 41:43 41:52 41:58   64/64: 33:30 33:35 33:41 32:46
//   32 requests, a window of 512, 64 / 80 / 96 rows            192/128: 41:39 42:46 42:51          128/128: 30:26 30:32 30:34         64/64: 25:24 26:29 26:31
// Where there are few keys in all its fixed cost loses: one request of 300 tokens, 64 to 128 rows, 22:12, 21:11 and 18:10.
constexpr int kChunkRows = 80;

// records in flight; at first the requests' units are held there
static size_t ring_bytes(int dk, int dv) {
  return std::max<size_t>((size_t)kC4Warps * kC4Stages * ((dk + dv) / kGroupDims) * kRecBytesPerGroup, kHeldBytes);
}

int cache4_grid(const Cache4Args& a, int rows, int per_sm) {
  const long long tiles = a.n_sel ? (long long)a.N * ((a.hpg + rows - 1) / rows) : ((long long)a.N * a.hpg + rows - 1) / rows + a.S;
  const long long units = tiles * a.G * (a.n_sel ? a.n_sel : std::max(a.P, 1));
  return (int)std::min<long long>(per_sm * 148, std::max<long long>(units, 1));
}

template <typename T, class Core>
static size_t core_workspace(const Cache4Args& a) {
  return split_bytes(cache4_grid(a, Core::kRows, Core::kBlocksPerSm), Core::kRows, a.dv);
}
template <typename T, class Core>
static int launch_core(const Cache4Args& a, const char* name, cudaStream_t st) {
  auto kern = cache4_attn_kernel<T, Core>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kC4Smem);
  if (e != cudaSuccess) return fail(NSA_ERR_LAUNCH, "cache4_attn: cannot reserve shared memory: %s", cudaGetErrorString(e));
  const int blocks = cache4_grid(a, Core::kRows, Core::kBlocksPerSm);
  {
    KernelTimer kt(name, st);
    kern<<<blocks, kC4Threads, ring_bytes(a.dk, a.dv) + Core::extra_smem(a.dk), st>>>(a);
    if (int rc = check_launch("cache4_attn")) return rc;
  }
  return launch_combine(a, blocks, Core::kRows, sizeof(T) == 4, st);
}

// the tensor-core kernels load and store their rows 16 bytes at a time
static bool mma_aligned(const Cache4Args& a) { return (uintptr_t)a.q % 16 == 0 && (uintptr_t)a.out % 16 == 0 && a.sq_tok % 8 == 0 && a.sq_head % 8 == 0; }

#define NSA_C4_FMA(FN, ...)                                                                              \
  (dtype == NSA_F32 ? (a.dv > 128 ? FN<float, FmaCore<float, kFmaRows, 8>>(__VA_ARGS__)                  \
                                  : FN<float, FmaCore<float, kFmaRows, 4>>(__VA_ARGS__))                 \
                    : (a.dv > 128 ? FN<__nv_bfloat16, FmaCore<__nv_bfloat16, kFmaRows, 8>>(__VA_ARGS__)  \
                                  : FN<__nv_bfloat16, FmaCore<__nv_bfloat16, kFmaRows, 4>>(__VA_ARGS__)))
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
  NSA_REQUIRE(std::isfinite(d->scale), "cache4_attn: scale %g is not finite", (double)d->scale);
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

extern "C" NSA_API int nsa_cache4_setup(void) {
  if (!fa_timeout_counter()) return fail(NSA_ERR_LAUNCH, "cache4_setup: cannot set up the time-out record of this device");
  return NSA_OK;
}

extern "C" NSA_API size_t nsa_cache4_attn_workspace_bytes(const nsa_cache4_desc* desc) {
  Cache4Args a;
  if (cache4_args(desc, a) != NSA_OK || a.N == 0 || a.S == 0) return 0;
  const int dtype = desc->dtype;
  const size_t fma = NSA_C4_FMA(core_workspace, a);
  if (dtype != NSA_BF16 || !cache4_mma_dims(a)) return fma;
  return std::max({fma, cache4_mma_workspace(a), a.n_sel ? 0 : cache4_chunk_workspace(a)});
}

extern "C" NSA_API int nsa_cache4_attn_fwd(const nsa_cache4_desc* desc, void* workspace, size_t workspace_bytes, void* stream) {
  Cache4Args a;
  if (int rc = cache4_args(desc, a)) return rc;
  if (a.N == 0 || a.S == 0) return NSA_OK;
  NSA_REQUIRE(a.table_ld >= a.P, "cache4_attn: table rows %lld apart overlap, they have %d pages", (long long)a.table_ld, a.P);
  NSA_REQUIRE(a.q && a.starts && a.lengths && a.out && a.L && a.M && (a.P == 0 || a.table) && (a.n_pages == 0 || a.cache) &&
                  (a.n_sel == 0 || a.indices), "cache4_attn: null pointer");
  NSA_REQUIRE((uintptr_t)a.cache % 16 == 0, "cache4_attn: the cache must be 16-byte aligned");
  const size_t need = nsa_cache4_attn_workspace_bytes(desc);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
    return fail(NSA_ERR_WORKSPACE, "cache4_attn: needs %zu bytes of 16-byte aligned scratch, got %zu", need, workspace_bytes);
  a.ws = (uint8_t*)workspace;
  cudaStream_t st = (cudaStream_t)stream;
  const int dtype = desc->dtype;
  if (dtype == NSA_BF16 && cache4_mma_dims(a) && mma_aligned(a)) {
    // Each request goes to the kernel that suits its rows, by their numbers on the device.  One launch is enough where no request can have many
    // rows, or where as many tokens as the requests' bounds allow say that all have: lengths on the device may be less, so the kernel for many
    // rows then takes every request there is.
    const int most = desc->max_new > 0 ? std::min(desc->max_new, a.N) : a.N;
    if (a.n_sel || (int64_t)most * a.hpg < kChunkRows) return launch_mma(a, st);
    if (desc->max_new > 0 && (int64_t)a.S * desc->max_new <= a.N) return launch_chunk(a, st);
    a.rows_lo = kChunkRows;
    if (int rc = launch_chunk(a, st)) return rc;
    a.rows_lo = 0;
    a.rows_hi = kChunkRows;
    return launch_mma(a, st);
  }
  return NSA_C4_FMA(launch_core, a, "cache4_attn_fma", st);
}
