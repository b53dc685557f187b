// Block tables of a step, and keys and values into and out of the 4-bit paged cache.
#include "cache4.cuh"

namespace nsa {

// ------------------------------------------------------------------------------------------------ block tables
constexpr int kTblThreads = 256;
constexpr int kTblMaxRequests = 16384;                      // two prefix sums of this many requests fit in shared memory
constexpr int kTblSmem = 2 * (kTblMaxRequests + 1) * 4;
constexpr int kTblTokensPerBlock = 2048;

struct TablesArgs {
  const int32_t *cached, *fresh, *free_pages;
  int32_t* table;
  int64_t table_ld;
  int64_t* slots;
  int32_t *positions, *starts, *lengths, *pages;
  int S, P, F, N, page;
};

// Lengths and sums of them are held below 2^30, whatever the caller's numbers: no index derived from them leaves 32 bits.
__device__ __forceinline__ int bounded(int x) { return min(max(x, 0), 1 << 29); }
__device__ __forceinline__ int add(int x, int y) { return min(x + y, 1 << 30); }

// Every block forms the prefix sums of all requests' new tokens and new pages (8 bytes a request out of L2, far less than what a
// second launch or a wait between blocks costs), then deals with its own 2048 tokens.  A token whose position opens a page takes
// that page off the free list and writes it into the table; old entries are only read, so no two threads touch one place.
// Bound by the launch and two dependent reads.
__global__ void __launch_bounds__(kTblThreads) block_tables_kernel(const TablesArgs a) {
  extern __shared__ int32_t sm_tbl[];
  int32_t* first_tok = sm_tbl;                  // [S + 1]
  int32_t* first_page = sm_tbl + a.S + 1;       // [S + 1]
  __shared__ int2 warp_sum[kTblThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 run = make_int2(0, 0);
  for (int base = 0; base < a.S; base += kTblThreads) {
    const int r = base + threadIdx.x;
    int2 x = make_int2(0, 0);
    int len = 0;
    if (r < a.S) {
      const int c = bounded(a.cached[r]);
      x.x = bounded(a.fresh[r]);
      len = c + x.x;
      x.y = (len + a.page - 1) / a.page - (c + a.page - 1) / a.page;
    }
    int2 s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int2 y = make_int2(__shfl_up_sync(0xffffffffu, s.x, o), __shfl_up_sync(0xffffffffu, s.y, o));
      if (lane >= o) { s.x = add(s.x, y.x); s.y = add(s.y, y.y); }
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int2 before = run;
    for (int w = 0; w < kTblThreads / 32; ++w) {
      const int2 t = warp_sum[w];
      if (w < warp) { before.x = add(before.x, t.x); before.y = add(before.y, t.y); }
      run.x = add(run.x, t.x);
      run.y = add(run.y, t.y);
    }
    if (r < a.S) {
      first_tok[r] = before.x + s.x - x.x;
      first_page[r] = before.y + s.y - x.y;
      if (blockIdx.x == 0) {
        a.starts[r] = first_tok[r];
        a.lengths[r] = len;
      }
    }
  }
  if (threadIdx.x == 0) {
    first_tok[a.S] = run.x;
    if (blockIdx.x == 0) {
      a.starts[a.S] = run.x;
      a.pages[0] = run.y;
    }
  }
  __syncthreads();
  const int lo = blockIdx.x * kTblTokensPerBlock, hi = min(a.N, lo + kTblTokensPerBlock);
  for (int i = lo + threadIdx.x; i < hi; i += kTblThreads) {
    if (i >= run.x) {
      a.slots[i] = -1;
      a.positions[i] = -1;
      continue;
    }
    int r = 0, up = a.S;                        // last request that starts at or before i and is not empty
    while (up - r > 1) {
      const int mid = (r + up) >> 1;
      if (first_tok[mid] <= i) r = mid; else up = mid;
    }
    const int c = bounded(a.cached[r]), pos = c + i - first_tok[r], pi = pos / a.page, off = pos - pi * a.page;
    const int have = (c + a.page - 1) / a.page;
    int id = -1;
    if (pi < a.P) {
      if (pi < have) {
        id = a.table[(int64_t)r * a.table_ld + pi];
      } else {
        const int at = first_page[r] + pi - have;
        id = at < a.F ? a.free_pages[at] : -1;
        if (off == 0) a.table[(int64_t)r * a.table_ld + pi] = id;
      }
    }
    a.slots[i] = id < 0 ? -1 : (int64_t)id * a.page + off;
    a.positions[i] = pos;
  }
}

// ------------------------------------------------------------------------------------------------ tokens into pages
// x rounded to the nearest whole number of steps of y, exactly: a quotient that 32 bits round onto k + 1/2 is settled by the sign of
// x - (k + 1/2) y, which an fma has exact as long as y has few significant bits; true ties go to the even one.
__device__ __forceinline__ float nearest_multiple(float x, float y) {
  const float t = __fdiv_rn(x, y), f = floorf(t);
  if (t - f != 0.5f) return rintf(t);
  const float d = fmaf(-t, y, x);
  return d > 0.f ? f + 1.f : d < 0.f ? f : rintf(t);
}

// a seventh of `a` to 8 significant bits (multiples of 2^-24 at the low end): what fp16 holds exactly
__device__ __forceinline__ float scale_of(float a) {
  const float t = __fdiv_rn(a, 7.f);
  const int e = max((int)(__float_as_uint(t) >> 23) - 127 - 7, -24);      // (a power of two that t was rounded up to gives the same scale)
  const float u = __uint_as_float((uint32_t)(e + 127) << 23);
  return nearest_multiple(a, 7.f * u) * u;                                // 7 u: three bits
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t stride, bool wide, float (&x)[8]) {
  if (wide) {
    if constexpr (sizeof(T) == 2) {
      const uint4 w = *reinterpret_cast<const uint4*>(p);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 w = reinterpret_cast<const float4*>(p)[i];
        x[4 * i] = w.x; x[4 * i + 1] = w.y; x[4 * i + 2] = w.z; x[4 * i + 3] = w.w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elem<T>::ld(p + i * stride);
  }
}

struct StoreArgs {
  const void *k, *v;
  int64_t sk[3], sv[3];        // strides (token, group, dimension)
  const int64_t* slots;
  uint8_t* cache;
  int64_t n_slots;
  int N, G, gk, gv;
  bool wide_k, wide_v;
};

// One warp per (token, group), four lanes per 32 dimensions: each holds eight, the largest magnitude goes round the four.  Values
// are written as 16-bit pieces of four dimensions of one token, so the four lanes first exchange their words.
template <typename T>
__global__ void __launch_bounds__(128) cache4_append_kernel(const StoreArgs a) {
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (int64_t)a.N * a.G) return;
  const int tok = (int)(item / a.G), g = (int)(item % a.G), lane = threadIdx.x & 31, j = lane & 3, quad0 = lane & ~3;
  const int64_t slot = a.slots[tok];
  if (slot < 0 || slot >= a.n_slots) return;
  const int groups = a.gk + a.gv, key = (int)(slot % kRecTokens);
  uint8_t* rec = a.cache + (slot / kPageTokens * a.G + g) * ((int64_t)kRecsPerPage * groups * kRecBytesPerGroup) +
                 slot % kPageTokens / kRecTokens * (groups * kRecBytesPerGroup);
  const int t = key >> 3, n = key & 7, pair = n >> 1, odd = n & 1;
  for (int c0 = 0; c0 < groups; c0 += 8) {
    const int c = c0 + (lane >> 2);
    float x[8] = {};
    if (c < a.gk)
      load8((const T*)a.k + tok * a.sk[0] + g * a.sk[1] + (c * kGroupDims + 8 * j) * a.sk[2], a.sk[2], a.wide_k, x);
    else if (c < groups)
      load8((const T*)a.v + tok * a.sv[0] + g * a.sv[1] + ((c - a.gk) * kGroupDims + 8 * j) * a.sv[2], a.sv[2], a.wide_v, x);
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -kMaxHeld), kMaxHeld);      // the cache holds finite numbers only
      m = fmaxf(m, fabsf(x[i]));
    }
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const float s = scale_of(m);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float k = s > 0.f ? fminf(fmaxf(nearest_multiple(x[i], s), -7.f), 7.f) : 0.f;
      w |= (uint32_t)((int)k + 8) << (4 * i);
    }
    uint32_t we[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) we[e] = __shfl_sync(0xffffffffu, w, quad0 + e);
    if (c >= groups) continue;
    uint8_t* chunk = rec + c * kChunkBytes;
    if (c < a.gk) {
      *reinterpret_cast<uint32_t*>(chunk + (n * 4 + j) * 8 + t * 4) = w;
    } else {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int d = 2 * j + b;
        uint32_t h = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) h |= ((we[e] >> (4 * d)) & 15u) << (4 * e);
        *reinterpret_cast<uint16_t*>(chunk + (d * 4 + pair) * 8 + (2 * t + odd) * 2) = (uint16_t)h;
      }
    }
    if (j == 0) *reinterpret_cast<__half*>(rec + groups * kChunkBytes + c * kChunkScaleBytes + (4 * pair + 2 * t + odd) * 2) = __float2half_rn(s);
  }
}

// ------------------------------------------------------------------------------------------------ and back
struct LoadArgs {
  void *k, *v;                 // [N, G, dk], [N, G, dv] contiguous
  const int64_t* slots;
  const uint8_t* cache;
  int64_t n_slots;
  int N, G, gk, gv;
};

template <typename T>
__global__ void __launch_bounds__(128) cache4_read_kernel(const LoadArgs a) {
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (int64_t)a.N * a.G) return;
  const int tok = (int)(item / a.G), g = (int)(item % a.G), lane = threadIdx.x & 31, j = lane & 3;
  const int64_t slot = a.slots[tok];
  const bool held = slot >= 0 && slot < a.n_slots;
  const int groups = a.gk + a.gv, key = (int)(held ? slot % kRecTokens : 0);
  const uint8_t* rec = a.cache + (held ? (slot / kPageTokens * a.G + g) * ((int64_t)kRecsPerPage * groups * kRecBytesPerGroup) +
                                             slot % kPageTokens / kRecTokens * (groups * kRecBytesPerGroup) : 0);
  const int t = key >> 3, n = key & 7, pair = n >> 1, odd = n & 1;
  for (int c = lane >> 2; c < groups; c += 8) {
    alignas(16) T x[8];
    uint32_t w = 0x88888888u;
    float s = 0.f;
    if (held) {
      const uint8_t* chunk = rec + c * kChunkBytes;
      s = __half2float(*reinterpret_cast<const __half*>(rec + groups * kChunkBytes + c * kChunkScaleBytes + (4 * pair + 2 * t + odd) * 2));
      if (c < a.gk) {
        w = *reinterpret_cast<const uint32_t*>(chunk + (n * 4 + j) * 8 + t * 4);
      } else {
        w = 0;
#pragma unroll
        for (int d = 0; d < 8; ++d)
          w |= (((uint32_t)*reinterpret_cast<const uint16_t*>(chunk + (d * 4 + pair) * 8 + (2 * t + odd) * 2) >> (4 * j)) & 15u) << (4 * d);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) Elem<T>::st(&x[i], (float)((int)((w >> (4 * i)) & 15u) - 8) * s);
    T* to = c < a.gk ? (T*)a.k + item * (a.gk * kGroupDims) + c * kGroupDims + 8 * j
                     : (T*)a.v + item * (a.gv * kGroupDims) + (c - a.gk) * kGroupDims + 8 * j;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(x)[i];
  }
}

static int check_cache(const char* who, const void* cache, int n_pages, int G, int dk, int dv) {
  NSA_REQUIRE(n_pages >= 0 && G > 0, "%s: bad page or group count %d/%d", who, n_pages, G);
  NSA_REQUIRE(dk > 0 && dv > 0 && dk <= kMaxHeadDim && dv <= kMaxHeadDim && dk % kGroupDims == 0 && dv % kGroupDims == 0,
              "%s: head dims %d/%d are no multiples of %d up to %d", who, dk, dv, kGroupDims, kMaxHeadDim);
  NSA_REQUIRE((uintptr_t)cache % 16 == 0, "%s: the cache must be 16-byte aligned", who);
  return NSA_OK;
}

static bool wide_ok(const void* p, const int64_t* s, size_t esize) {
  const int64_t m = 16 / (int64_t)esize;
  return (uintptr_t)p % 16 == 0 && s[2] == 1 && s[0] % m == 0 && s[1] % m == 0;
}

}  // namespace nsa

using namespace nsa;

extern "C" NSA_API size_t nsa_cache4_page_bytes(int dk, int dv) {
  if (dk <= 0 || dv <= 0 || dk > kMaxHeadDim || dv > kMaxHeadDim || dk % kGroupDims || dv % kGroupDims) return 0;
  return (size_t)page_bytes(dk, dv);
}

extern "C" NSA_API int nsa_block_tables(const int32_t* cached, const int32_t* fresh, int32_t* table, int64_t table_ld, const int32_t* free_pages,
                                        int64_t* slots, int32_t* positions, int32_t* starts, int32_t* lengths, int32_t* pages, int S, int P,
                                        int F, int N, int page, void* stream) {
  NSA_REQUIRE(S >= 0 && P >= 0 && F >= 0 && N >= 0 && table_ld >= P, "block_tables: bad sizes %d/%d/%d/%d", S, P, F, N);
  NSA_REQUIRE(S <= kTblMaxRequests, "block_tables: %d requests, at most %d in one call", S, kTblMaxRequests);
  NSA_REQUIRE(page > 0 && page <= 65536, "block_tables: page size %d outside 1..65536", page);
  NSA_REQUIRE(starts && pages && (S == 0 || (cached && fresh && lengths)) && (S == 0 || P == 0 || table) && (F == 0 || free_pages) &&
                  (N == 0 || (slots && positions)), "block_tables: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = cudaFuncSetAttribute(block_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTblSmem);
  if (e != cudaSuccess) return fail(NSA_ERR_LAUNCH, "block_tables: cannot reserve shared memory: %s", cudaGetErrorString(e));
  const TablesArgs a{cached, fresh, free_pages, table, table_ld, slots, positions, starts, lengths, pages, S, P, F, N, page};
  KernelTimer kt("block_tables", st);
  block_tables_kernel<<<N > 0 ? (N + kTblTokensPerBlock - 1) / kTblTokensPerBlock : 1, kTblThreads, 2 * (S + 1) * 4, st>>>(a);
  return check_launch("block_tables");
}

extern "C" NSA_API int nsa_cache4_append(const void* k, const void* v, const int64_t* strides6, const int64_t* slots, void* cache, int N, int n_pages,
                                         int G, int dk, int dv, int dtype, void* stream) {
  if (int rc = check_cache("cache4_append", cache, n_pages, G, dk, dv)) return rc;
  NSA_REQUIRE(N >= 0 && (int64_t)N * G <= 0x7fffffffll, "cache4_append: %d tokens of %d groups", N, G);
  NSA_REQUIRE(dtype == NSA_F32 || dtype == NSA_BF16, "cache4_append: unsupported dtype %d", dtype);
  if (N == 0 || n_pages == 0) return NSA_OK;
  NSA_REQUIRE(k && v && strides6 && slots && cache, "cache4_append: null pointer");
  const size_t es = dtype == NSA_F32 ? 4 : 2;
  StoreArgs a{k, v, {}, {}, slots, (uint8_t*)cache, (int64_t)n_pages * kPageTokens, N, G, dk / kGroupDims, dv / kGroupDims,
              wide_ok(k, strides6, es), wide_ok(v, strides6 + 3, es)};
  for (int i = 0; i < 3; ++i) { a.sk[i] = strides6[i]; a.sv[i] = strides6[3 + i]; }
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = (unsigned)(((int64_t)N * G + 3) / 4);
  KernelTimer kt("cache4_append", st);
  if (dtype == NSA_F32) cache4_append_kernel<float><<<grid, 128, 0, st>>>(a);
  else cache4_append_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(a);
  return check_launch("cache4_append");
}

extern "C" NSA_API int nsa_cache4_read(const void* cache, const int64_t* slots, void* k, void* v, int N, int n_pages, int G, int dk, int dv, int dtype,
                                       void* stream) {
  if (int rc = check_cache("cache4_read", cache, n_pages, G, dk, dv)) return rc;
  NSA_REQUIRE(N >= 0 && (int64_t)N * G <= 0x7fffffffll, "cache4_read: %d tokens of %d groups", N, G);
  NSA_REQUIRE(dtype == NSA_F32 || dtype == NSA_BF16, "cache4_read: unsupported dtype %d", dtype);
  if (N == 0) return NSA_OK;
  NSA_REQUIRE(k && v && slots && (cache || n_pages == 0), "cache4_read: null pointer");
  NSA_REQUIRE((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, "cache4_read: outputs must be 16-byte aligned");
  const LoadArgs a{k, v, slots, (const uint8_t*)cache, (int64_t)n_pages * kPageTokens, N, G, dk / kGroupDims, dv / kGroupDims};
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = (unsigned)(((int64_t)N * G + 3) / 4);
  KernelTimer kt("cache4_read", st);
  if (dtype == NSA_F32) cache4_read_kernel<float><<<grid, 128, 0, st>>>(a);
  else cache4_read_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(a);
  return check_launch("cache4_read");
}
