// Attention over the 4-bit paged cache: how the work is cut up, shared by its kernels.
//
// A segment is what one softmax runs over for one tile of rows: (request, kv group, tile of ROWS rows), a row being one query token and
// one of the group's heads; in the selected form (token, kv group, tile).  Its units are pages of 64 keys (selected form: places of the
// token's block list).  The units of all segments, one after the other, are dealt to the thread blocks in equal shares, wherever the
// segments end: requests of any mixture of lengths keep every SM busy to the end.  A block merges what it has of a segment; a segment
// that one block has whole goes straight to the output, the others leave partial results (running maximum, sum and unnormalised
// output, 32 bits) that combine_kernel joins in order.  A block has at most two partial segments, its first and its last.  Nothing is
// known of the lengths on the host: every block forms the prefix sums over the requests for itself.
#pragma once
#include "cache4.cuh"

namespace nsa {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSelMax = 32;          // places of a block list: one per lane
// Requests whose units are held in shared memory at once.  A unit number has 64 bits: rows in tiles of 8 times up to 2^23 pages, a prompt
// of 371 000 tokens with 16 heads a group has 2^31 of them already.
constexpr int kHeldRequests = 4096, kHeldBytes = kHeldRequests * 8;

// Probabilities that become fp16 are 2^7 times what they are against a row's reference: the reference lags by 2^8 at most, so they stay below
// 65504, and fp16 ends at 2^-32 of the reference instead of 2^-25.  (Sums have the factor too; results take it out.)
constexpr float kProbShift = 7.f, kProbUnshift = 0.0078125f;
// An exponent is one multiply-add, x c2 - (m c2): rounding the product in brackets moves all of a row's by the same 2^-25 of it, which cancels.
// From here on it would be places of its own (and fp16 overflow): x - m comes first then, and is exact where it matters.
constexpr float kFarLogit = 0x1p20f;       // log2 units

struct Segment {
  int tok0;        // first token of the request among the step's (selected form: the token)
  int row0, nrows; // first flattened row (token * heads per group + head) within the request and how many there are
  int r, g;
  int pos0;        // position of token tok0
  int lo, hi;      // units
};

// what a block leaves about its last segment, if the segment starts there and ends in a later block
struct SplitRecord {
  int pieces;                        // blocks that have a part of it, this one the first; 0: there is no such segment
  int tok0, row0, nrows, g, pad[3];
};

// a / b of numbers that are not negative; nearly always both have 32 bits, and dividing those takes a quarter of the instructions
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return ((unsigned long long)(a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

// Block c of n has units [share(c), share(c + 1)) of total; with fewer units than blocks the first ones have one each.
__device__ __forceinline__ long long share(long long total, int c, int n) {
  n = (int)min((long long)n, total);
  return c >= n ? total : quotient(total * c, n);
}
__device__ __forceinline__ int block_of(long long total, long long u, int n) {
  n = (int)min((long long)n, total);
  return (int)quotient((u + 1) * n - 1, total);               // the last c with total * c / n <= u
}

// KEYS: keys of a unit (one page, or two).  OVER: what starting and ending a segment costs, in units, when shares are dealt: they count
// as units behind the segment's own, and a block whose share of a segment is only of those does nothing for it.
// SEL: the selected form can be asked for.
template <int ROWS, int KEYS, int OVER, bool SEL>
struct Walk {
  static constexpr int kChunk = kHeldRequests;
  const Cache4Args& a;
  Segment s;
  int tile, tiles, len, fresh;              // of the current request (selected form: fresh is the first request's first token)
  long long total;

  __device__ Walk(const Cache4Args& args) : a(args) {}

  // the walk's place, to lie in shared memory while a kernel needs its registers
  struct Place {
    Segment s;
    int tile, tiles, len, fresh, place;
    long long u, end, total;
  };
  __device__ __forceinline__ void save(Place& p, long long u, long long end, int place) const { p = Place{s, tile, tiles, len, fresh, place, u, end, total}; }
  __device__ __forceinline__ void restore(const Place& p, long long& u, long long& end, int& place) {
    s = p.s; tile = p.tile; tiles = p.tiles; len = p.len; fresh = p.fresh; total = p.total;
    u = p.u; end = p.end; place = p.place;
  }

  __device__ __forceinline__ int row_tiles(int n) const { return (n * a.hpg + ROWS - 1) / ROWS; }
  __device__ __forceinline__ int length() const { return s.hi - s.lo + OVER; }
  // tokens and length of a request: nothing outside [0, N] whatever the arrays hold
  __device__ __forceinline__ void request(int r, int& tok0, int& n, int& length) const {
    const int b = min(max(a.starts[r], 0), a.N), e = min(max(a.starts[r + 1], 0), a.N);
    tok0 = b;
    n = max(e - b, 0);
    if (n * a.hpg < a.rows_lo || n * a.hpg >= a.rows_hi) n = 0;
    length = min(max(a.lengths[r], 0), 1 << 30);
  }
  // units that some row of tile t can see (at least one, so that every row is written)
  __device__ __forceinline__ void bounds(int length, int n, int t, int& lo, int& hi) const {
    const int p0 = length - n;
    const int first = p0 + t * ROWS / a.hpg, last = p0 + min(n * a.hpg - 1, t * ROWS + ROWS - 1) / a.hpg;
    hi = last < 0 ? 0 : min(last / KEYS + 1, (a.P * kPageTokens + KEYS - 1) / KEYS);
    lo = a.window > 0 ? max(first - a.window + 1, 0) / KEYS : 0;
    if (hi <= lo) { lo = 0; hi = 1; }
  }

  __device__ __forceinline__ void set_tile() {
    s.row0 = tile * ROWS;
    if (SEL && a.n_sel) {
      s.nrows = min(ROWS, a.hpg - s.row0);
      return;
    }
    s.nrows = min(ROWS, fresh * a.hpg - s.row0);
    bounds(len, fresh, tile, s.lo, s.hi);
  }
  __device__ __forceinline__ void set_request(int r) {
    s.r = r;
    request(r, s.tok0, fresh, len);
    s.pos0 = len - fresh;
    tiles = row_tiles(fresh);
  }
  // selected form: request and position of token s.tok0, given that it belongs to s.r or a later one
  __device__ __forceinline__ void set_token() {
    while (s.r + 1 < a.S && a.starts[s.r + 1] <= s.tok0) ++s.r;
    s.pos0 = a.lengths[s.r] - a.starts[s.r + 1] + s.tok0;
  }

  // units (of one group) of requests base .. base + kChunk - 1 into shared memory: a thread per request, or where a request has many
  // tiles a warp
  template <int T>
  __device__ __forceinline__ void fill(int base, long long* held) const {
    const int n = min(kChunk, a.S - base), lane = threadIdx.x & 31;
    if ((long long)a.N * a.hpg <= 4ll * ROWS * a.S) {
      for (int i = threadIdx.x; i < n; i += T) {
        int tok0, fresh, length;
        long long sum = 0;
        request(base + i, tok0, fresh, length);
        for (int t = 0, m = row_tiles(fresh); t < m; ++t) {
          int lo, hi;
          bounds(length, fresh, t, lo, hi);
          sum += hi - lo + OVER;
        }
        held[i] = sum;
      }
    } else {
      for (int i = threadIdx.x >> 5; i < n; i += T / 32) {
        int tok0, fresh, length;
        long long sum = 0;
        request(base + i, tok0, fresh, length);
        for (int t = lane, m = row_tiles(fresh); t < m; t += 32) {
          int lo, hi;
          bounds(length, fresh, t, lo, hi);
          sum += hi - lo + OVER;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) held[i] = sum;
      }
    }
    __syncthreads();
  }

  // Number of all units; all T threads of the block take part.  scratch: T / 32 + 3 long longs of shared memory, held: kHeldBytes of it.
  template <int T>
  __device__ __forceinline__ void start(long long* scratch, long long* held) {
    if (SEL && a.n_sel) {
      fresh = min(max(a.starts[0], 0), a.N);
      const int n = max(min(a.starts[a.S], a.N) - fresh, 0);
      tiles = (a.hpg + ROWS - 1) / ROWS;
      s.lo = 0;
      s.hi = a.n_sel;
      total = (long long)n * a.G * tiles * length();
      return;
    }
    long long x = 0;
    for (int base = 0; base < a.S; base += kChunk) {
      if (base) __syncthreads();
      fill<T>(base, held);
      for (int i = threadIdx.x; i < min(kChunk, a.S - base); i += T) x += held[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    total = 0;
    for (int w = 0; w < T / 32; ++w) total += scratch[w];
    total *= a.G;
    __syncthreads();
  }
  // Segment that unit u (< total) lies in; returns its place within the segment.
  template <int T>
  __device__ __forceinline__ int seek(long long u, long long* scratch, long long* held) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (SEL && a.n_sel) {
      const long long seg = quotient(u, length()), of_tiles = quotient(seg, tiles), of_groups = quotient(of_tiles, a.G);
      tile = (int)(seg - of_tiles * tiles);
      s.g = (int)(of_tiles - of_groups * a.G);
      s.tok0 = fresh + (int)of_groups;
      int lo = 0, up = a.S;                     // last request that starts at or before the token: 32 probes at a time
      while (up - lo > 1) {
        const int step = (up - lo + 31) / 32, at = lo + lane * step;
        const unsigned le = __ballot_sync(0xffffffffu, at < up && a.starts[at < up ? at : lo] <= s.tok0);
        const int k = max(31 - __clz(le), 0);
        up = min(up, lo + (k + 1) * step);
        lo += k * step;
      }
      s.r = lo;
      set_token();
      set_tile();
      return (int)(u - seg * length());
    }
    long long run = 0;
    bool found = false;
    for (int base = 0; base < a.S && !found; base += kChunk) {
      if (a.S > kChunk) {
        __syncthreads();
        fill<T>(base, held);
      }
      for (int i0 = 0; i0 < min(kChunk, a.S - base) && !found; i0 += T) {
        const int i = i0 + threadIdx.x;
        const long long x = i < min(kChunk, a.S - base) ? held[i] * a.G : 0;
        long long p = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long y = __shfl_up_sync(0xffffffffu, p, o);
          if (lane >= o) p += y;
        }
        __syncthreads();
        if (lane == 31) scratch[warp] = p;
        if (threadIdx.x == 0) scratch[T / 32] = -1;
        __syncthreads();
        long long before = run;
        for (int w = 0; w < T / 32; ++w) {
          if (w < warp) before += scratch[w];
          run += scratch[w];
        }
        p += before;
        if (u >= p - x && u < p) {
          scratch[T / 32] = base + i;
          scratch[T / 32 + 1] = u - (p - x);
          scratch[T / 32 + 2] = held[i];
        }
        __syncthreads();
        found = scratch[T / 32] >= 0;
      }
    }
    set_request((int)scratch[T / 32]);
    const long long off = scratch[T / 32 + 1], per = scratch[T / 32 + 2];
    __syncthreads();
    s.g = (int)quotient(off, per);
    long long place = off - s.g * per;
    for (int t0 = 0;; t0 += 32) {               // 32 tiles at a time
      int lo, hi, p = 0;
      if (t0 + lane < tiles) {
        bounds(len, fresh, t0 + lane, lo, hi);
        p = hi - lo + OVER;
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, p, o);
        if (lane >= o) p += y;
      }
      const unsigned past = __ballot_sync(0xffffffffu, p > place);
      if (past || t0 + 32 >= tiles) {
        const int k = past ? __ffs(past) - 1 : tiles - 1 - t0;
        if (k > 0) place -= __shfl_sync(0xffffffffu, p, k - 1);
        tile = t0 + k;
        set_tile();
        return (int)place;
      }
      place -= __shfl_sync(0xffffffffu, p, 31);
    }
  }
  // Unit at which block c's share begins.  A boundary inside a segment that is short against a share moves to the segment's nearer end: what
  // such a segment would cost as two partial results is more than the shares then differ by.  Leaves the walk at that unit, its place in `place`.
  template <int T>
  __device__ __forceinline__ long long boundary(int c, int n, long long* scratch, long long* held, int& place) {
    long long u = share(total, c, n);
    place = 0;
    if (u >= total) return u;
    place = seek<T>(u, scratch, held);
    if (place > 0 && 4ll * length() * n <= total) {
      const bool up = 2 * place >= length();
      u += up ? length() - place : -place;
      place = 0;
      if (up && u < total) next();
    }
    return u;
  }
  // the segment after this one (there is one)
  __device__ __forceinline__ void next() {
    if (++tile < tiles) return set_tile();
    tile = 0;
    if (++s.g < a.G) return set_tile();
    s.g = 0;
    if (SEL && a.n_sel) {
      ++s.tok0;
      set_token();
      return set_tile();
    }
    for (int r0 = s.r + 1; r0 < a.S; r0 += 32) {          // 32 requests at a time: other launches may own long runs of them
      const int r = r0 + (threadIdx.x & 31);
      int tok0, n = 0, length;
      if (r < a.S) request(r, tok0, n, length);
      const unsigned some = __ballot_sync(0xffffffffu, n > 0);
      if (some) {
        set_request(r0 + __ffs(some) - 1);
        return set_tile();
      }
    }
  }
};

// Workspace: records of all blocks, then two partial results a block: [rows][dv] unnormalised outputs, [rows] (maximum, sum).
__host__ __device__ __forceinline__ size_t split_rec_bytes(int blocks) { return ((size_t)blocks * sizeof(SplitRecord) + 255) / 256 * 256; }
__host__ __device__ __forceinline__ size_t split_part_floats(int rows, int dv) { return (size_t)rows * (dv + 2); }
__host__ __device__ __forceinline__ size_t split_bytes(int blocks, int rows, int dv) {
  return split_rec_bytes(blocks) + (size_t)blocks * 2 * split_part_floats(rows, dv) * 4;
}
__device__ __forceinline__ float* split_part(const Cache4Args& a, int blocks, int rows, int block, int which) {
  return reinterpret_cast<float*>(a.ws + split_rec_bytes(blocks)) + ((size_t)block * 2 + which) * split_part_floats(rows, a.dv);
}

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// A query row with a NaN or an infinity has no softmax: it is NaN from the start (each kernel's), so are all its logits and the sum of its
// probabilities.  The maximum is not (the larger of a number and NaN is the number) and follows here, or the row would pass for one that sees nothing.
__device__ __forceinline__ float max_of_row(float m, float l) { return l == l ? m : CUDART_NAN_F; }

// row i of a segment: its token and head
__device__ __forceinline__ int64_t out_row(const Cache4Args& a, const Segment& s, int i) {
  const int f = s.row0 + i;
  return (int64_t)(s.tok0 + f / a.hpg) * a.H + s.g * a.hpg + f % a.hpg;
}

// the tensor-memory kernel for many rows a request (cache4_chunk.cu)
size_t cache4_chunk_workspace(const Cache4Args& a);
int launch_chunk(const Cache4Args& a, cudaStream_t st);

// bf16 queries on mma.sync (cache4_mma.cu)
bool cache4_mma_dims(const Cache4Args& a);
size_t cache4_mma_workspace(const Cache4Args& a);
int launch_mma(const Cache4Args& a, cudaStream_t st);

// thread blocks of a launch: what the device holds at once, or as many as there can be units
int cache4_grid(const Cache4Args& a, int rows, int per_sm);
int launch_combine(const Cache4Args& a, int blocks, int rows, bool f32, cudaStream_t st);

}  // namespace nsa
