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
  static constexpr int kRows = RT;
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
template <typename T, class Core>
__global__ void __launch_bounds__(kC4Threads) cache4_attn_kernel(const Cache4Args a) {
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

// Joins the partial results of one row of one split segment: block (owner, row).  The pieces are the owner's last segment and the first
// segments of the blocks after it; four warps take every fourth of them, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(128) cache4_combine_kernel(const Cache4Args a, int blocks, int rows) {
  const SplitRecord rec = reinterpret_cast<const SplitRecord*>(a.ws)[blockIdx.x];
  const int r = blockIdx.y;
  if (!rec.open || r >= rec.nrows) return;
  __shared__ float acc[4][kMaxHeadDim];
  __shared__ float2 ml[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // the last block that has a unit of the segment
  int last = blockIdx.x;
  {
    int lo = blockIdx.x, up = blocks;
    while (up - lo > 1) {
      const int mid = (lo + up) >> 1;
      if (share(rec.total, mid, blocks) < rec.last) lo = mid; else up = mid;
    }
    last = lo;
  }
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

int launch_combine(const Cache4Args& a, int blocks, int rows, bool f32, cudaStream_t st) {
  KernelTimer kt("cache4_combine", st);
  const dim3 grid(blocks, rows);
  if (f32) cache4_combine_kernel<float><<<grid, 128, 0, st>>>(a, blocks, rows);
  else cache4_combine_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(a, blocks, rows);
  return check_launch("cache4_combine");
}

int cache4_sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
  return n;
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int kFmaRows = 8;
constexpr int kFmaSmem = 227 * 1024 - 4096;
constexpr int kFmaBlocksPerSm = 2;

static size_t ring_bytes(int dk, int dv) { return (size_t)kC4Warps * kC4Stages * ((dk + dv) / kGroupDims) * kRecBytesPerGroup; }

static int fma_blocks(const Cache4Args& a) {
  // no more blocks than units there can be
  const long long tiles = a.n_sel ? (long long)a.N * ((a.hpg + kFmaRows - 1) / kFmaRows) : ((long long)a.N * a.hpg + kFmaRows - 1) / kFmaRows + a.S;
  const long long units = tiles * a.G * (a.n_sel ? a.n_sel : std::max(a.P, 1));
  return (int)std::min<long long>(kFmaBlocksPerSm * 148, std::max<long long>(units, 1));
}

template <typename T, int GV>
static int launch_fma(const Cache4Args& a, cudaStream_t st) {
  using Core = FmaCore<T, kFmaRows, GV>;
  auto kern = cache4_attn_kernel<T, Core>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFmaSmem);
  if (e != cudaSuccess) return fail(NSA_ERR_LAUNCH, "cache4_attn: cannot reserve shared memory: %s", cudaGetErrorString(e));
  const int blocks = fma_blocks(a);
  {
    KernelTimer kt("cache4_attn_fma", st);
    kern<<<blocks, kC4Threads, ring_bytes(a.dk, a.dv) + Core::extra_smem(a.dk), st>>>(a);
    if (int rc = check_launch("cache4_attn")) return rc;
  }
  return launch_combine(a, blocks, kFmaRows, sizeof(T) == 4, st);
}

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
  return split_bytes(fma_blocks(a), kFmaRows, a.dv);
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
  const bool wide = a.dv > 128;
  if (desc->dtype == NSA_F32) return wide ? launch_fma<float, 8>(a, st) : launch_fma<float, 4>(a, st);
  return wide ? launch_fma<__nv_bfloat16, 8>(a, st) : launch_fma<__nv_bfloat16, 4>(a, st);
}
