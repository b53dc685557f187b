// Block tables of a step, and keys and values into and out of the 4-bit paged cache.
#include "cache4.cuh"

namespace nsa {

// ------------------------------------------------------------------------------------------------ block tables
constexpr int kTblMaxThreads = 512;
constexpr int kTblMaxRequests = 16384;                      // two prefix sums of this many requests fit in shared memory
constexpr int kTblSmem = 2 * (kTblMaxRequests + 1) * 4;
constexpr int kTblTokensPerBlock = 512;

struct TablesArgs {
  const int32_t *cached, *fresh, *free_pages;
  int32_t* table;
  int64_t table_ld;
  int64_t* slots;
  int32_t *positions, *starts, *lengths, *pages;
  int S, P, F, N, page;
};

// Lengths are held to 2^29 and sums of them below 2^30, whatever the caller's numbers.  So two sums add up within 32 bits, a sum is never less
// than its last term, and (first_tok[0] being 0) a token's request starts at or before it: positions, and page numbers in a row or on the
// free list, are not negative.
__device__ __forceinline__ int bounded(int x) { return min(max(x, 0), 1 << 29); }
__device__ __forceinline__ int add(int x, int y) { return min(x + y, (1 << 30) - 1); }

// Every block forms the prefix sums of all requests' new tokens and new pages (8 bytes a request out of L2, far less than what a
// second launch or a wait between blocks costs), then deals with its own 512 tokens.  A token whose position opens a page takes
// that page off the free list and writes it into the table; old entries are only read, so no two threads touch one place.
// Bound by the launch and dependent reads (the sums, a search per token, the table): 3.1 us for 256 requests of one token, 4.8 us for 45 000
// tokens of 1000 requests (7.3 us with 2048 tokens a block).  512 threads take half the steps over many requests (with 256 the second case
// takes 5.9 us), up to 256 requests they only cost their start (the first case 3.4 us).
__global__ void __launch_bounds__(kTblMaxThreads) block_tables_kernel(const TablesArgs a) {
  extern __shared__ int32_t sm_tbl[];
  int32_t* first_tok = sm_tbl;                  // [S + 1]
  int32_t* first_page = sm_tbl + a.S + 1;       // [S + 1]
  __shared__ int2 warp_sum[kTblMaxThreads / 32];
  const int threads = blockDim.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 run = make_int2(0, 0);
  for (int base = 0; base < a.S; base += threads) {
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
    for (int w = 0; w < threads / 32; ++w) {
      const int2 t = warp_sum[w];
      if (w < warp) { before.x = add(before.x, t.x); before.y = add(before.y, t.y); }
      run.x = add(run.x, t.x);
      run.y = add(run.y, t.y);
    }
    if (r < a.S) {
      first_tok[r] = add(before.x, s.x) - x.x;
      first_page[r] = add(before.y, s.y) - x.y;
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
  for (int i = lo + threadIdx.x; i < hi; i += threads) {
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
        const unsigned at = (unsigned)first_page[r] + (unsigned)(pi - have);      // (below 2^30 + 2^29 + 2^30)
        id = at < (unsigned)a.F ? a.free_pages[at] : -1;
        if (off == 0) a.table[(int64_t)r * a.table_ld + pi] = id;
      }
    }
    a.slots[i] = id < 0 ? -1 : (int64_t)id * a.page + off;
    a.positions[i] = pos;
  }
}

// ------------------------------------------------------------------------------------------------ tokens into pages
// x over step rounded to the nearest whole number c, ties to the even one, exactly, as the bits of 1.5 * 2^23 + c: the reciprocal's product is
// off by less than one, and the remainder x - c step is exact (c step has 12 bits at most, the difference no more places than x), so it
// says whether c is the nearest.  (For an odd c a remainder of just a half is too much already: the limit is one place lower.)
__device__ __forceinline__ int nearest_bits(float x, float step, float inv, float half) {
  const float r = fmaf(x, inv, 12582912.f);
  const float d = fmaf(12582912.f - r, step, x);
  int bits = __float_as_int(r);
  if (fabsf(d) > __int_as_float(__float_as_int(half) - (bits & 1))) bits += (__float_as_int(d) >> 31) | 1;
  return bits;
}
constexpr int kWholeBits = 0x4b400000;               // 1.5 * 2^23

// a seventh of `a` to 8 significant bits (multiples of 2^-24 at the low end): what fp16 holds exactly
__device__ __forceinline__ float scale_of(float a) {
  const float t = a * 0.142857142857f;
  // (next to a power of two, the one above or below it as the unit gives the same scale)
  const int e = max((int)(__float_as_uint(t) >> 23) - 127 - 7, -24);
  const float u = __uint_as_float((uint32_t)(e + 127) << 23), inv_u = __uint_as_float((uint32_t)(127 - e) << 23);
  return (float)(nearest_bits(a, 7.f * u, 0.142857142857f * inv_u, 3.5f * u) - kWholeBits) * u;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t stride, bool wide, float (&x)[8]) {
  if (wide) {
    if constexpr (sizeof(T) == 2) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 w = __ldg(reinterpret_cast<const float4*>(p) + i);
        x[4 * i] = w.x; x[4 * i + 1] = w.y; x[4 * i + 2] = w.z; x[4 * i + 3] = w.w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elem<T>::ld(p + i * stride);
  }
}

// ------------------------------------------------------------------------------------------------
// A block has 16 tokens of one group.  Tokens of a prompt sit in consecutive slots, and the 16 slots of a record that are all among a
// call's tokens, one after the other, are dealt with together: the block that has the first of them takes the whole record through shared
// memory, so that it is read or written in 16-byte pieces.  Other tokens go straight to their bytes.  Four lanes have 32 dimensions of a
// token, eight each; consecutive lanes have consecutive dimensions.
// ------------------------------------------------------------------------------------------------
constexpr int kTokThreads = 256;

struct TokenList {
  int n, first;                  // how many; index of the record's first token in the call, or -1
  int token[32];
  long long slot[32];
};

__device__ __forceinline__ void build_list(const int64_t* slots, int N, int64_t n_slots, TokenList& list) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, t0 = blockIdx.x * kRecTokens - 15;          // places 0..46: the block's tokens are 15..30
    const int i0 = t0 + lane, i1 = i0 + 32;
    const long long s0 = i0 >= 0 && i0 < N ? slots[i0] : -1, s1 = lane < 16 && i1 < N ? slots[i1] : -1;
    const bool ok0 = s0 >= 0 && s0 < n_slots, ok1 = s1 >= 0 && s1 < n_slots;
    const long long wrap = __shfl_sync(0xffffffffu, s1, 0);
    long long up0 = __shfl_down_sync(0xffffffffu, s0, 1), up1 = __shfl_down_sync(0xffffffffu, s1, 1);
    if (lane == 31) up0 = wrap;
    const uint64_t follows = (uint64_t)__ballot_sync(0xffffffffu, ok0 && up0 == s0 + 1) | (uint64_t)__ballot_sync(0xffffffffu, ok1 && up1 == s1 + 1) << 32;
    const uint32_t starts = __ballot_sync(0xffffffffu, ok0 && s0 % kRecTokens == 0 && (follows >> lane & 0x7fffu) == 0x7fffu);   // whole records by their first place
    const uint32_t mine = starts & 0x7fff8000u;                               // (never two: they are 16 places apart)
    const int lead = mine ? __ffs(mine) - 1 : -1;
    // places 15..45 by lane
    const int place = lane + 15, i = t0 + place;
    const long long s_hi = __shfl_sync(0xffffffffu, s1, (place - 32) & 31), s_lo = __shfl_sync(0xffffffffu, s0, min(place, 31));
    const long long slot = place < 32 ? s_lo : s_hi;
    const bool valid = place < 46 && i < N;
    const int from = slot >= 0 ? place - (int)(slot % kRecTokens) : -1;
    const bool covered = valid && slot >= 0 && slot < n_slots && from >= 0 && from < 32 && (starts >> from & 1);
    const bool take = valid && ((place <= 30 && !covered) || (lead >= 0 && covered && from == lead));
    const uint32_t who = __ballot_sync(0xffffffffu, take);
    if (take) {
      const int at = __popc(who & ((1u << lane) - 1u));
      list.token[at] = i;
      list.slot[at] = slot;
    }
    if (lane == 0) {
      list.n = __popc(who);
      list.first = lead < 0 ? -1 : t0 + lead;
    }
  }
  __syncthreads();
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

// where slot's record of group g begins
__device__ __forceinline__ int64_t record_at(int64_t slot, int g, int G, int groups) {
  return (slot / kPageTokens * G + g) * (int64_t)(kRecsPerPage * groups * kRecBytesPerGroup) + (int)(slot & (kPageTokens - 1)) / kRecTokens * (groups * kRecBytesPerGroup);
}

// codes and scales of chunks c0 .. c1 - 1 of a record
__device__ __forceinline__ void copy_chunks(uint4* to, const uint4* from, int groups, int c0, int c1) {
  constexpr int kCodes = kChunkBytes / 16, kScales = kChunkScaleBytes / 16;
  const int n = (c1 - c0) * kCodes, m = (c1 - c0) * kScales;
  for (int i = threadIdx.x; i < n + m; i += kTokThreads) {
    const int at = i < n ? c0 * kCodes + i : groups * kCodes + c0 * kScales + i - n;
    to[at] = from[at];
  }
}

// chunks c0 .. c1 - 1 of the list's tokens, all of the keys or all of the values (V): the lanes of a warp do the same thing
template <typename T, bool V>
__device__ __forceinline__ void append_chunks(const StoreArgs& a, const TokenList& list, uint8_t* staged, int g, int c0, int c1) {
  const int groups = a.gk + a.gv, quad0 = threadIdx.x & 28, cn = c1 - c0, items = list.n * cn * 4;
  const unsigned over = (65536u + cn - 1) / max(cn, 1);         // idx / cn = idx * over >> 16 for idx (cn - 1) < 65536
  const T* src = V ? (const T*)a.v + g * a.sv[1] - a.gk * kGroupDims * a.sv[2] : (const T*)a.k + g * a.sk[1];
  const int64_t s_tok = V ? a.sv[0] : a.sk[0], s_dim = V ? a.sv[2] : a.sk[2];
  const bool wide = V ? a.wide_v : a.wide_k;
#pragma unroll 2
  for (int base = 0; base < items; base += kTokThreads) {
    const int item = base + threadIdx.x, idx = item >> 2, e = (int)((unsigned)idx * over >> 16), c = c0 + idx - e * cn, j = item & 3;
    const bool on = item < items;
    const int tok = on ? list.token[e] : 0;
    const long long slot = on ? list.slot[e] : -1;
    float x[8] = {};
    if (on) load8(src + tok * s_tok + (c * kGroupDims + 8 * j) * s_dim, s_dim, wide, x);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float m = __uint_as_float(top);
    if (top > 0x475f2000u) {             // 57120: the cache holds finite numbers only (the four lanes agree)
      m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -kMaxHeld), kMaxHeld);
        m = fmaxf(m, fabsf(x[i]));
      }
      m = fmaxf(m, __shfl_xor_sync(0xfu << quad0, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xfu << quad0, m, 2));
    }
    const float s = scale_of(m), inv = s > 0.f ? __frcp_rn(s) : 0.f, half = s > 0.f ? 0.5f * s : CUDART_INF_F;
    int code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) code[i] = nearest_bits(x[i], s, inv, half);
    if (__any_sync(0xffffffffu, s < 0x1p-16f)) {         // a scale of few places may be a good deal below a seventh
#pragma unroll
      for (int i = 0; i < 8; ++i) code[i] = min(max(code[i], kWholeBits - 7), kWholeBits + 7);
    }
    uint32_t w = 0;                                      // sum of (c + 8) 16^i
#pragma unroll
    for (int i = 7; i >= 0; --i) w = w * 16 + (uint32_t)code[i];
    w -= (uint32_t)(kWholeBits - 8) * 0x11111111u;
    uint32_t we[4];                      // values lie as four dimensions 8 apart: the four lanes exchange their words
    if (V) {
#pragma unroll
      for (int i = 0; i < 4; ++i) we[i] = __shfl_sync(0xffffffffu, w, quad0 + i) >> (8 * j);
    }
    if (slot < 0 || slot >= a.n_slots) continue;
    const int key = (int)slot & (kRecTokens - 1), t = key >> 3, n = key & 7, pair = n >> 1, odd = n & 1;
    uint8_t* rec = list.first >= 0 && tok >= list.first && tok < list.first + kRecTokens ? staged : a.cache + record_at(slot, g, a.G, groups);
    uint8_t* chunk = rec + c * kChunkBytes;
    if (!V) {
      *reinterpret_cast<uint32_t*>(chunk + (n * 4 + j) * 8 + t * 4) = w;
    } else {
      // dimensions n = 2 j and 2 j + 1 of the four lanes, a nibble each
      const uint32_t lo = (we[0] & 15u) | (we[1] & 15u) << 4 | (we[2] & 15u) << 8 | (we[3] & 15u) << 12;
      const uint32_t hi = (we[0] >> 4 & 15u) | (we[1] & 0xf0u) | (we[2] & 0xf0u) << 4 | (we[3] & 0xf0u) << 8;
      uint8_t* to = chunk + (8 * j + pair) * 8 + (2 * t + odd) * 2;
      *reinterpret_cast<uint16_t*>(to) = (uint16_t)lo;
      *reinterpret_cast<uint16_t*>(to + 32) = (uint16_t)hi;
    }
    if (j == 0) *reinterpret_cast<__half*>(rec + groups * kChunkBytes + c * kChunkScaleBytes + (4 * pair + 2 * t + odd) * 2) = __float2half_rn(s);
  }
}

template <typename T>
__global__ void __launch_bounds__(kTokThreads) cache4_append_kernel(const StoreArgs a) {
  __shared__ TokenList list;
  __shared__ __align__(16) uint8_t staged[2 * kMaxHeadDim / kGroupDims * kRecBytesPerGroup];
  const int g = blockIdx.y, groups = a.gk + a.gv;
  const int c0 = blockIdx.z * groups / gridDim.z, c1 = (blockIdx.z + 1) * groups / gridDim.z;      // this block's chunks
  build_list(a.slots, a.N, a.n_slots, list);
  append_chunks<T, false>(a, list, staged, g, c0, min(c1, a.gk));
  append_chunks<T, true>(a, list, staged, g, max(c0, a.gk), c1);
  if (list.first < 0) return;
  __syncthreads();
  uint4* to = reinterpret_cast<uint4*>(a.cache + record_at(a.slots[list.first], g, a.G, groups));
  copy_chunks(to, reinterpret_cast<const uint4*>(staged), groups, c0, c1);
}

// ------------------------------------------------------------------------------------------------ and back
struct LoadArgs {
  void *k, *v;                 // [N, G, dk], [N, G, dv] contiguous
  const int64_t* slots;
  const uint8_t* cache;
  int64_t n_slots;
  int N, G, gk, gv;
};

template <typename T, bool V>
__device__ __forceinline__ void read_chunks(const LoadArgs& a, const TokenList& list, const uint8_t* staged, int g, int c0, int c1) {
  const int groups = a.gk + a.gv, cn = c1 - c0, items = list.n * cn * 4;
  const unsigned over = (65536u + cn - 1) / max(cn, 1);
  for (int item = threadIdx.x; item < items; item += kTokThreads) {
    const int idx = item >> 2, e = (int)((unsigned)idx * over >> 16), c = c0 + idx - e * cn, j = item & 3, tok = list.token[e];
    const long long slot = list.slot[e];
    alignas(16) T x[8];
    uint32_t w = 0x88888888u;
    float s = 0.f;
    if (slot >= 0 && slot < a.n_slots) {
      const int key = (int)slot & (kRecTokens - 1), t = key >> 3, n = key & 7, pair = n >> 1, odd = n & 1;
      const uint8_t* rec = list.first >= 0 && tok >= list.first && tok < list.first + kRecTokens ? staged : a.cache + record_at(slot, g, a.G, groups);
      const uint8_t* chunk = rec + c * kChunkBytes;
      s = __half2float(*reinterpret_cast<const __half*>(rec + groups * kChunkBytes + c * kChunkScaleBytes + (4 * pair + 2 * t + odd) * 2));
      if (!V) {
        w = *reinterpret_cast<const uint32_t*>(chunk + (n * 4 + j) * 8 + t * 4);
      } else {
        w = 0;
#pragma unroll
        for (int d = 7; d >= 0; --d)
          w = w << 4 | (((uint32_t)*reinterpret_cast<const uint16_t*>(chunk + (d * 4 + pair) * 8 + (2 * t + odd) * 2) >> (4 * j)) & 15u);
      }
    }
    const float s8 = -8.f * s;           // (c - 8) s without a rounding: c s has 12 bits
#pragma unroll
    for (int i = 0; i < 8; ++i) Elem<T>::st(&x[i], fmaf((float)((w >> (4 * i)) & 15u), s, s8));
    const int64_t row = (int64_t)tok * a.G + g;
    T* to = V ? (T*)a.v + row * (a.gv * kGroupDims) + (c - a.gk) * kGroupDims + 8 * j : (T*)a.k + row * (a.gk * kGroupDims) + c * kGroupDims + 8 * j;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(x)[i];
  }
}

template <typename T>
__global__ void __launch_bounds__(kTokThreads) cache4_read_kernel(const LoadArgs a) {
  __shared__ TokenList list;
  __shared__ __align__(16) uint8_t staged[2 * kMaxHeadDim / kGroupDims * kRecBytesPerGroup];
  const int g = blockIdx.y, groups = a.gk + a.gv;
  const int c0 = blockIdx.z * groups / gridDim.z, c1 = (blockIdx.z + 1) * groups / gridDim.z;
  build_list(a.slots, a.N, a.n_slots, list);
  if (list.first >= 0) {
    const uint4* from = reinterpret_cast<const uint4*>(a.cache + record_at(a.slots[list.first], g, a.G, groups));
    copy_chunks(reinterpret_cast<uint4*>(staged), from, groups, c0, c1);
    __syncthreads();
  }
  read_chunks<T, false>(a, list, staged, g, c0, min(c1, a.gk));
  read_chunks<T, true>(a, list, staged, g, max(c0, a.gk), c1);
}

// Blocks of 16 tokens; few of them are cut up further by chunks, until there are two for every SM.
static dim3 token_grid(int N, int G, int groups) {
  const int64_t blocks = (int64_t)((N + kRecTokens - 1) / kRecTokens) * G;
  const int cut = (int)((2 * 148 + blocks - 1) / blocks);
  return dim3((N + kRecTokens - 1) / kRecTokens, G, cut < 1 ? 1 : cut > groups ? groups : cut);
}

static int check_cache(const char* who, const void* cache, int n_pages, int G, int dk, int dv) {
  NSA_REQUIRE(n_pages >= 0 && G > 0 && G <= 65535, "%s: bad page or group count %d/%d", who, n_pages, G);
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
  NSA_REQUIRE(N <= 1 << 30, "block_tables: %d tokens, at most %d in one call", N, 1 << 30);
  NSA_REQUIRE(S <= kTblMaxRequests, "block_tables: %d requests, at most %d in one call", S, kTblMaxRequests);
  NSA_REQUIRE(page > 0 && page <= 65536, "block_tables: page size %d outside 1..65536", page);
  NSA_REQUIRE(starts && pages && (S == 0 || (cached && fresh && lengths)) && (S == 0 || P == 0 || table) && (F == 0 || free_pages) &&
                  (N == 0 || (slots && positions)), "block_tables: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = cudaFuncSetAttribute(block_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTblSmem);
  if (e != cudaSuccess) return fail(NSA_ERR_LAUNCH, "block_tables: cannot reserve shared memory: %s", cudaGetErrorString(e));
  const TablesArgs a{cached, fresh, free_pages, table, table_ld, slots, positions, starts, lengths, pages, S, P, F, N, page};
  KernelTimer kt("block_tables", st);
  block_tables_kernel<<<N > 0 ? (N + kTblTokensPerBlock - 1) / kTblTokensPerBlock : 1, S <= 256 ? 256 : kTblMaxThreads, 2 * (S + 1) * 4, st>>>(a);
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
  const dim3 grid = token_grid(N, G, (dk + dv) / kGroupDims);
  KernelTimer kt("cache4_append", st);
  if (dtype == NSA_F32) cache4_append_kernel<float><<<grid, kTokThreads, 0, st>>>(a);
  else cache4_append_kernel<__nv_bfloat16><<<grid, kTokThreads, 0, st>>>(a);
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
  const dim3 grid = token_grid(N, G, (dk + dv) / kGroupDims);
  KernelTimer kt("cache4_read", st);
  if (dtype == NSA_F32) cache4_read_kernel<float><<<grid, kTokThreads, 0, st>>>(a);
  else cache4_read_kernel<__nv_bfloat16><<<grid, kTokThreads, 0, st>>>(a);
  return check_launch("cache4_read");
}
