// Chunks of many new tokens over the 4-bit paged cache on 5th-generation tensor cores (tcgen05 + TMEM).
//
// A block owns 256 rows (query token, head) of one kv group in two MMA tiles of 128 and walks the keys 128 at a time (two pages).  Roles (512 threads):
//   warps 0-3 / 4-7  softmax of tile 0 / 1, one row per thread: they also bring the row's queries in (fp16, scaled to a largest magnitude
//                    in [2^14, 2^15) by a power of two) and write its output
//   warps 8-11       unpack a tile's keys and values out of L2 into shared memory: fp16 holds (c - 8) s exactly
//   warp 13          walks the block's segments and hands the pieces to the others
//   warp 12          issues the MMAs: S_i = Q_i K^T (both operands in shared memory), O_i += P_i V (P in tensor memory)
// TMEM columns and the order PV0(j) QK0(j+1) PV1(j) QK1(j+1) are those of the dense forward kernel.  Probabilities are rounded to fp16:
// by 2^-11 down to 2^-21 of the row's reference, by 2^-32 of the reference below (kProbShift).  Those of the first 64 keys are handed over while
// the others are formed (head dims 128/128: 1080 -> 1035 us, 192/128: no change).
//
// Where a code lies in its word fixes in which order a thread unpacks it for free; the two operands of a product only have to agree.  So
// eight dimensions of a query and a key lie in the order 0 4 1 5 2 6 3 7, and dimension 8 e + n of a group of 32 values is column
// 8 (n / 2) + 2 e + n % 2 of the output tile, put back in order when the row is written.
//
// Bound by the round trip of a tile: softmax about 2100 clocks (1024 of them the exponentials of 128 keys alone, shared with the other tile's
// warps), its own two products 1280 at head dims 192/128, handing over on either side of both 400 to 900; about 4400 clocks for two tiles of
// 128 keys, where the tensor pipe needs 2560.  2000 new tokens behind 30000 earlier ones, 16 query heads a group, 4 groups: 2.1 ms (1200 TFLOP/s)
// on a chip that is not warm; a long loop of it is slowed by the power limit (2.3 to 2.5 ms).
#include <algorithm>

#include "attn_args.cuh"
#include "cache4_attn.cuh"
#include "fa_sm100.cuh"
#include "sm100_ptx.cuh"

namespace nsa {

using namespace ptx;

constexpr int kChM = 128, kChN = 128, kChRows = 256, kChThreads = 512;
constexpr int kChRegsSoftmax = 168, kChRegsUnpack = 112, kChRegsIssue = 64;
constexpr int kChRegsNeeded = (256 * kChRegsSoftmax + 128 * kChRegsUnpack + 128 * kChRegsIssue + kChThreads - 1) / kChThreads;   // per thread at launch
constexpr int kChOver = 2;           // see Walk
constexpr float kChGrow = 8.f;       // log2 units

template <int DK, int DV>
struct ChunkSmem {
  static constexpr int kQBytes = kChM * DK * 2, kKBytes = kChN * DK * 2, kVBytes = kChN * DV * 2;
  static constexpr int oQ = 0, oK = oQ + 2 * kQBytes, oV = oK + kKBytes, oOut = oV + 2 * kVBytes, oBar = oOut + 8 * 2048;
  static constexpr int kDynamic = oBar + 768 + 1024;       // slack to align the base to the swizzle atom
};

// units [p0, p0 + n) of a segment, as one warp finds them and the roles take them; n = 0 ends the list
struct ChunkPiece {
  int tok0, row0, nrows, r, g, pos0, p0, n, whole, part;
};
constexpr int kChPieces = 4, kChRoleWarps = 13;

struct ChunkBarriers {
  uint64_t piece_full[kChPieces], piece_empty[kChPieces];
  ChunkPiece piece[kChPieces];
  uint64_t q_full[2], k_full, k_empty, v_full[2], v_empty[2], s_full[2], p_half[2], p_full[2], pv_done[2], o_free[2], drained;
  long long scratch[kChThreads / 32 + 3];
  uint32_t tmem_base;
  int abort;
};

// fp16 x fp16 -> fp32, dense
constexpr uint32_t idesc_f16(int M, int N, int a_mn_major, int b_mn_major) {
  return (1u << 4) | ((uint32_t)a_mn_major << 15) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t code_bits(uint32_t x, uint32_t mask) {      // (x & mask) | 1024 in both halves
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, 0x64006400, 0xEA;" : "=r"(r) : "r"(x), "r"(mask));
  return r;
}
// 32 lanes x 8 consecutive 32-bit columns (the rescaling has few registers to spare beside a row's logits)
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// The issuing warp's instructions, carried out where `on` says so
__device__ __forceinline__ void mma_ss(uint32_t on, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t on, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(on)
      : "memory");
}
// four codes of each half of a word, nibble by nibble, times the half's scale
__device__ __forceinline__ uint4 unpack8(uint32_t w, __half2 s) {
  const __half2 bias = __float2half2_rn(-1032.f), sixteenth = __float2half2_rn(0.0625f), bias16 = __float2half2_rn(-72.f);
  const uint32_t v = w >> 8;
  uint4 r;
  r.x = h2u(__hmul2(__hadd2(u2h(code_bits(w, 0x000f000fu)), bias), s));
  r.y = h2u(__hmul2(__hfma2(u2h(code_bits(w, 0x00f000f0u)), sixteenth, bias16), s));
  r.z = h2u(__hmul2(__hadd2(u2h(code_bits(v, 0x000f000fu)), bias), s));
  r.w = h2u(__hmul2(__hfma2(u2h(code_bits(v, 0x00f000f0u)), sixteenth, bias16), s));
  return r;
}

template <int DK, int DV>
__global__ void __launch_bounds__(kChThreads, 1) cache4_chunk_kernel(const Cache4Args a, int* timeouts) {
  using SM = ChunkSmem<DK, DV>;
  constexpr int GK = DK / kGroupDims, GV = DV / kGroupDims, kRecBytes = (GK + GV) * kRecBytesPerGroup;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  ChunkBarriers* bar = reinterpret_cast<ChunkBarriers*>(smem + SM::oBar);
  volatile int* abort = &bar->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->q_full[i], 128);
      mbar_init(&bar->v_full[i], 128);
      mbar_init(&bar->v_empty[i], 1);
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->p_half[i], 128);
      mbar_init(&bar->p_full[i], 128);
      mbar_init(&bar->pv_done[i], 1);
      mbar_init(&bar->o_free[i], 128);
    }
    for (int i = 0; i < kChPieces; ++i) {
      mbar_init(&bar->piece_full[i], 1);
      mbar_init(&bar->piece_empty[i], kChRoleWarps);
    }
    mbar_init(&bar->k_full, 128);
    mbar_init(&bar->k_empty, 1);
    mbar_init(&bar->drained, 1);
    bar->abort = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 12) tmem_alloc(&bar->tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_base;

  Walk<kChRows, kChN, kChOver, false> walk(a);
  long long* held = reinterpret_cast<long long*>(smem);       // where queries will be
  walk.template start<kChThreads>(bar->scratch, held);
  // once any block has given up on a wait the device's results are void: later blocks skip their work
  if (threadIdx.x == 0) bar->scratch[0] = *(volatile const int*)timeouts != 0 ? 0 : walk.total;
  __syncthreads();
  walk.total = bar->scratch[0];
  __syncthreads();
  int place0 = 0;
  long long begin = 0, end = 0;
#pragma unroll 1
  for (int c = 1; c >= 0; --c) {          // (one copy of the code: what runs once costs its fetching)
    end = begin;
    begin = walk.template boundary<kChThreads>(blockIdx.x + c, gridDim.x, bar->scratch, held, place0);
  }
  __syncthreads();
  // piece number c of the block into registers, its place free again; a wait that runs out reads as the end of the list
  auto take = [&](int c) {
    ChunkPiece w;
    if (mbar_wait_warp(&bar->piece_full[c % kChPieces], (c / kChPieces) & 1, abort)) {
      w = bar->piece[c % kChPieces];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->piece_empty[c % kChPieces]);
    } else {
      w.n = 0;
    }
    return w;
  };
  auto pages_of = [&](const ChunkPiece& w, int unit, int& id0, int& id1) {
    id0 = 2 * unit < a.P ? a.table[w.r * a.table_ld + 2 * unit] : -1;
    id1 = 2 * unit + 1 < a.P ? a.table[w.r * a.table_ld + 2 * unit + 1] : -1;
    if (id0 >= a.n_pages) id0 = -1;
    if (id1 >= a.n_pages) id1 = -1;
  };

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kChRegsIssue));
    if (warp == 13) {
      // ---------------------------------------------------------- the block's pieces
      SplitRecord out{};
      long long u = begin;
      int place = place0;
      for (int c = 0;; ++c) {
        ChunkPiece w{};
        while (u < end && w.n <= 0) {
          const Segment& s = walk.s;
          const int share_n = (int)min((long long)(walk.length() - place), end - u);
          w = ChunkPiece{s.tok0, s.row0, s.nrows, s.r, s.g, s.pos0, s.lo + place, min(share_n, s.hi - s.lo - place), 0, place == 0};
          w.whole = place == 0 && w.n == s.hi - s.lo;
          if (place == 0 && !w.whole)
            out = SplitRecord{block_of(walk.total, u + s.hi - s.lo - 1, gridDim.x) - (int)blockIdx.x + 1, s.tok0, s.row0, s.nrows, s.g, {}};
          u += share_n;
          place = 0;
          if (u < end) walk.next();
        }
        if (w.n < 0) w.n = 0;        // the share ended among what ending a segment counts for
        if (!mbar_wait_warp(&bar->piece_empty[c % kChPieces], ((c / kChPieces) & 1) ^ 1, abort)) break;
        if (lane == 0) {
          bar->piece[c % kChPieces] = w;
          mbar_arrive(&bar->piece_full[c % kChPieces]);
        }
        if (w.n == 0) break;
      }
      if (lane == 0) reinterpret_cast<SplitRecord*>(a.ws)[blockIdx.x] = out;
    } else if (warp == 12) {
      // ---------------------------------------------------------- MMA issuer (warp-uniform loops, one elected lane issues)
      // One lane issues.  Up to 128 key dimensions the whole warp walks through the instructions, each carried out by its leader, and the code of
      // either tile is its own: the descriptors of 16 products cost fewer instructions so (head dims 128/128, 2048 tokens behind 30000: 934 us
      // against 1040 with a branch around them; prompts of up to 1500 tokens, whose starts fetch more code, 155 against 152).  With 192 the
      // branch and one copy of the code are faster: 2200 us against 2595.
      constexpr bool kBranch = DK > 128;
      constexpr int kCopies = kBranch ? 1 : 2;
      constexpr uint32_t idQK = idesc_f16(kChM, kChN, 0, 0), idPV = idesc_f16(kChM, DV, 0, 1);
      const uint64_t dQ0 = smem_desc_sw128(smem_u32(smem + SM::oQ), 16, 1024);
      const uint64_t dK0 = smem_desc_sw128(smem_u32(smem + SM::oK), 16, 1024);
      const uint64_t dV = smem_desc_sw128(smem_u32(smem + SM::oV), kChN * 128, 1024);
      const uint32_t leader = elect_one();
      auto by_leader = [&](auto&& f) {
        if constexpr (kBranch) {
          if (leader) f(1u);
          __syncwarp();
        } else {
          f(leader);
        }
      };
      auto issue_qk = [&](uint32_t on, int i) {
        const uint64_t dQ = desc_advance(dQ0, i * SM::kQBytes);
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk)
          mma_ss(on, tmem + i * 128, desc_advance(dQ, (kk >> 2) * (kChM * 128) + (kk & 3) * 32),
                 desc_advance(dK0, (kk >> 2) * (kChN * 128) + (kk & 3) * 32), idQK, kk > 0);
        commit(on, &bar->s_full[i]);
      };
      bool ok = true;
      int kc = 0, ic0 = 0, ic1 = 0, sc0 = 0, sc1 = 0;     // key tiles; segments and key tiles of either MMA tile so far
      for (int pc = 0; ok; ++pc) {
        const ChunkPiece w = take(pc);
        if (w.n == 0) break;
        const bool two = w.nrows > kChM;
        const int ntile = two ? 2 : 1;
        ok = mbar_wait_warp(&bar->q_full[0], ic0 & 1, abort) && (!two || mbar_wait_warp(&bar->q_full[1], ic1 & 1, abort)) &&
             mbar_wait_warp(&bar->k_full, kc & 1, abort);
        if (!ok) break;
        tc_fence_after();
        by_leader([&](uint32_t on) {
          issue_qk(on, 0);
          if (two) issue_qk(on, 1);
          commit(on, &bar->k_empty);
        });
        for (int j = 0; j < w.n && ok; ++j, ++kc) {
          const bool more = j + 1 < w.n;
          ok = mbar_wait_warp(&bar->v_full[kc & 1], (kc >> 1) & 1, abort);
#pragma unroll kCopies
          for (int i = 0; i < 2; ++i) {
            if (i >= ntile || !ok) break;
            ok = mbar_wait_warp(&bar->p_half[i], (i ? sc1 : sc0) & 1, abort);
            if (ok && j == 0) ok = mbar_wait_warp(&bar->o_free[i], ((i ? ic1 : ic0) & 1) ^ 1, abort);
            if (!ok) break;
            tc_fence_after();
            const uint64_t dv = desc_advance(dV, (kc & 1) * SM::kVBytes);
            auto issue_pv = [&](uint32_t on, int k0) {
#pragma unroll
              for (int kk = 0; kk < kChN / 32; ++kk)
                mma_ts(on, tmem + 256 + i * 128, tmem + i * 128 + (k0 + kk) * 8, desc_advance(dv, (k0 + kk) * 2048), idPV, j > 0 || k0 + kk > 0);
            };
            by_leader([&](uint32_t on) { issue_pv(on, 0); });
            ok = mbar_wait_warp(&bar->p_full[i], (i ? sc1 : sc0) & 1, abort);
            if (!ok) break;
            tc_fence_after();
            by_leader([&](uint32_t on) {
              issue_pv(on, kChN / 32);
              commit(on, &bar->pv_done[i]);
              if (i + 1 == ntile) commit(on, &bar->v_empty[kc & 1]);
            });
            if (more) {
              if (i == 0) {
                ok = mbar_wait_warp(&bar->k_full, (kc + 1) & 1, abort);
                if (!ok) break;
                tc_fence_after();
              }
              by_leader([&](uint32_t on) {
                issue_qk(on, i);
                if (i + 1 == ntile) commit(on, &bar->k_empty);
              });
            }
            if (i) ++sc1; else ++sc0;
          }
        }
        ++ic0;
        if (two) ++ic1;
      }
      if (__any_sync(0xffffffffu, *abort)) {        // products in flight end before the block gives its memory back, or another limit ends that
        volatile int overdue = 0;
        commit(leader, &bar->drained);
        mbar_wait_warp(&bar->drained, 0, &overdue);
      }
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------ keys and values: 4 bits in L2 -> fp16 in shared memory
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kChRegsUnpack));
    const int wq = warp - 8, n = lane >> 2, j = lane & 3;
    const uint32_t mine = n & 1 ? 0x3232 : 0x1010;       // of a pair of scales, this token's, twice
    const int vg = lane >> 4, vu = (lane >> 2) & 3;
    // keys: lane (n, j) holds 8 dimensions of tokens n and 8 + n; odd n take the odd group of a pair first, so that the eight lanes of a store
    // phase fill all eight 16-byte columns.  values: lane (group of a pair, dimensions n = 2 u and 2 u + 1, tokens 2 j, 2 j + 1, 8 + 2 j,
    // 8 + 2 j + 1).  A tile's keys are loaded while the tile before it is unpacked; there is time for the rest: keys wait for QK, values have two stages.
    uint2 kw[2][GK];
    ChunkPiece f;                  // piece and tile of the loads
    int ft = 0, pc = 0, id0 = -1, id1 = -1, id = -1;
    const uint8_t* src = nullptr;
    // the tile to load next, and its page: this warp's two records are half of one
    auto step = [&]() {
      if (++ft >= f.n) {
        f = take(pc++);
        ft = 0;
        if (f.n == 0) return;
        pages_of(f, f.p0, id0, id1);
      }
      id = wq < 2 ? id0 : id1;
      src = a.cache + (((int64_t)max(id, 0) * a.G + f.g) * kRecsPerPage + (wq & 1) * 2) * kRecBytes;
      if (ft + 1 < f.n) pages_of(f, f.p0 + ft + 1, id0, id1);
    };
    auto load_k = [&]() {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int g = 0; g < GK; ++g) {
          kw[r][g] = make_uint2(0, 0);
          if (id >= 0) kw[r][g] = __ldg(reinterpret_cast<const uint2*>(src + r * kRecBytes + (g ^ (n & 1)) * kChunkBytes + lane * 8));
        }
    };
    f.n = 0;
    step();
    if (f.n > 0) load_k();
    for (int kc = 0; f.n > 0; ++kc) {
      const int n0 = (f.p0 + ft) * kChN, maxpos = f.pos0 + (f.row0 + f.nrows - 1) / a.hpg, page = id;
      const int minlow = a.window > 0 ? f.pos0 + f.row0 / a.hpg - a.window + 1 : 0;
      const uint8_t* rec0 = src;
      uint2 ks[2][GK];               // four scales: tokens n with its neighbour, and 8 behind them
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int g = 0; g < GK; ++g) {
          ks[r][g] = make_uint2(0, 0);
          if (page >= 0)
            ks[r][g] = __ldg(reinterpret_cast<const uint2*>(rec0 + r * kRecBytes + (GK + GV) * kChunkBytes + (g ^ (n & 1)) * kChunkScaleBytes) + (n >> 1));
        }
      if (!mbar_wait_warp(&bar->k_empty, (kc & 1) ^ 1, abort)) break;
      uint8_t* sK = smem + SM::oK;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int g = 0; g < GK; ++g) {
          const int gg = g ^ (n & 1), row = (wq * 2 + r) * 16 + n;
          uint8_t* dst = sK + (g >> 1) * (kChN * 128) + row * 128 + ((((gg & 1) * 4 + j) ^ n) << 4);
          *reinterpret_cast<uint4*>(dst) = unpack8(kw[r][g].x, u2h(__byte_perm(ks[r][g].x, 0, mine)));
          *reinterpret_cast<uint4*>(dst + 8 * 128) = unpack8(kw[r][g].y, u2h(__byte_perm(ks[r][g].y, 0, mine)));
        }
      fence_proxy_async();
      mbar_arrive(&bar->k_full);
      step();
      if (f.n > 0) load_k();
      uint2 v0[2][GV / 2], v1[2][GV / 2], vs[2][GV / 2];
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int g = 0; g < GV / 2; ++g) {
          const uint8_t* rec = rec0 + r * kRecBytes;
          const uint2* c = reinterpret_cast<const uint2*>(rec + (GK + 2 * g + vg) * kChunkBytes);
          v0[r][g] = v1[r][g] = vs[r][g] = make_uint2(0, 0);
          if (page >= 0) {
            v0[r][g] = __ldg(c + 8 * vu + j);
            v1[r][g] = __ldg(c + 8 * vu + 4 + j);
            vs[r][g] = __ldg(reinterpret_cast<const uint2*>(rec + (GK + GV) * kChunkBytes + (GK + 2 * g + vg) * kChunkScaleBytes) + j);
          }
        }
      // what no row sees may never have been written: nothing of it enters, not as 0 times it either
      const bool edge = n0 + kChN - 1 > maxpos || n0 < minlow;
      if (!mbar_wait_warp(&bar->v_empty[kc & 1], ((kc >> 1) & 1) ^ 1, abort)) break;
      uint8_t* sV = smem + SM::oV + (kc & 1) * SM::kVBytes;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int g = 0; g < GV / 2; ++g) {
          uint8_t* dst = sV + g * (kChN * 128);
          const int rec0 = (wq * 2 + r) * 16;
#pragma unroll
          for (int q = 0; q < 4; ++q) {             // token 8 (q / 2) + 2 j + q % 2
            const int row = rec0 + 8 * (q >> 1) + 2 * j + (q & 1);
            const uint32_t x = q < 2 ? v0[r][g].x : v0[r][g].y, y = q < 2 ? v1[r][g].x : v1[r][g].y, z = q < 2 ? vs[r][g].x : vs[r][g].y;
            uint32_t sc = __byte_perm(z, z, q & 1 ? 0x3232 : 0x1010);
            if (edge && (n0 + row > maxpos || n0 + row < minlow)) sc = 0;
            *reinterpret_cast<uint4*>(dst + row * 128 + (((vg * 4 + vu) ^ (row & 7)) << 4)) =
                unpack8(__byte_perm(x, y, q & 1 ? 0x7632 : 0x5410), u2h(sc));
          }
        }
      fence_proxy_async();
      mbar_arrive(&bar->v_full[kc & 1]);
    }
  } else {
    // ------------------------------------------------------------ softmax and epilogue, one row per thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kChRegsSoftmax));
    const int i = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_base + i * 128, tO = tmem + lane_base + 256 + i * 128;
    float cl = 0.f;                      // logit of a unit of S
    int pos = -1, pos_next = -1;
    // The rows of a piece into shared memory: copied as they are while the last page of the piece before is worked on (its S has been read, so Q
    // is free), and turned into fp16 where they lie, a row a thread.  These loops run once a piece: they stay rolled, since what straight
    // code would save in instructions it loses many times over in fetching them.
    auto start_q = [&](const ChunkPiece& s) {
      const int f = s.row0 + i * kChM + r;
      const bool there = i * kChM + r < s.nrows;
      pos_next = there ? s.pos0 + f / a.hpg : -1;
      const int64_t off = there ? (s.tok0 + f / a.hpg) * a.sq_tok + (s.g * a.hpg + f % a.hpg) * a.sq_head : -1;
#pragma unroll 2
      for (int it = 0; it < DK / 8; ++it) {
        const int u = it * 32 + lane, row = u / (DK / 8), c = u % (DK / 8), rr = (warp & 3) * 32 + row;
        const int64_t at = __shfl_sync(0xffffffffu, off, row);
        const uint32_t dst = smem_u32(smem + SM::oQ + i * SM::kQBytes + (c >> 3) * (kChM * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"((const __nv_bfloat16*)a.q + max(at, (int64_t)0) + c * 8), "r"(at < 0 ? 0 : 16)
                     : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto finish_q = [&]() {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
      uint8_t* mine = smem + SM::oQ + i * SM::kQBytes + r * 128;
      uint32_t mx = 0;
#pragma unroll 4
      for (int c = 0; c < DK / 8; ++c) {
        const uint4 v = *reinterpret_cast<const uint4*>(mine + (c >> 3) * (kChM * 128) + (((c & 7) ^ (r & 7)) << 4));
        mx = __vmaxu2(__vmaxu2(mx, v.x & 0x7fff7fffu), __vmaxu2(__vmaxu2(v.y & 0x7fff7fffu, v.z & 0x7fff7fffu), v.w & 0x7fff7fffu));
      }
      mx = max(mx & 0xffffu, mx >> 16);
      const int k = mx ? min(14 - ((int)(mx >> 7) - 127), 100) : 0;
      // the scale's sign goes into the row, so that larger S is always the larger logit; scale 0 is a row of zeros
      const float up = mx >= 0x7f80 ? CUDART_NAN_F : __uint_as_float((uint32_t)(k + 127) << 23) * (a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : 0.f);
      cl = (a.scale == 0.f ? 1.f : fabsf(a.scale)) * __uint_as_float((uint32_t)(127 - k) << 23);
      pos = pos_next;
#pragma unroll 2
      for (int c = 0; c < DK / 8; ++c) {
        uint4* at = reinterpret_cast<uint4*>(mine + (c >> 3) * (kChM * 128) + (((c & 7) ^ (r & 7)) << 4));
        const uint4 v = *at;
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = __uint_as_float(w[e] << 16) * up;
          x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u) * up;
        }
        *at = make_uint4(h2u(__floats2half2_rn(x[0], x[4])), h2u(__floats2half2_rn(x[1], x[5])), h2u(__floats2half2_rn(x[2], x[6])), h2u(__floats2half2_rn(x[3], x[7])));
      }
      fence_proxy_async();
      mbar_arrive(&bar->q_full[i]);
    };
    bool ok = true;
    int sc = 0;                          // key tiles of earlier segments (barrier phases run on)
    int pc = 0;
    // Pieces stay in their places while this warp works on them, and are read there: registers are short beside a row's logits.
    auto release = [&](int c) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->piece_empty[c % kChPieces]);
    };
    // Moves pc on to the next piece that has rows for this tile: 1 there is one, 0 there is none, -1 (not waiting) it is not known yet.  A warp
    // that still has a piece's place must not wait for a later one: pieces without rows for its tile may fill all other places, and the
    // one it waits for would need this one's.
    auto find = [&](bool wait) {
      for (;; ++pc) {
        uint64_t* there = &bar->piece_full[pc % kChPieces];
        const uint32_t parity = (pc / kChPieces) & 1;
        if (wait) {
          if (!mbar_wait_warp(there, parity, abort)) return 0;
        } else if (!__all_sync(0xffffffffu, mbar_test(there, parity))) {
          return -1;
        }
        const ChunkPiece& w = bar->piece[pc % kChPieces];
        if (w.n == 0 || i * kChM < w.nrows) return w.n > 0 ? 1 : 0;
        release(pc);
      }
    };
    int next = -1;
    for (;;) {
      if (next < 0) {                    // (no piece is held here)
        next = find(true);
        if (next > 0) {
          start_q(bar->piece[pc % kChPieces]);
          finish_q();
        }
      }
      if (next <= 0) break;
      const int cur = pc;
      const ChunkPiece& s = bar->piece[cur % kChPieces];
      const int n = s.n, p0 = s.p0;
      const int row0 = s.row0 + i * kChM, my_pos = pos;
      // held within 2^-100 and 2^80, so that S (at most 2^39) times it is finite and -inf times it is -inf: beyond, values of S that differ at
      // all are worlds apart or all are one
      const float c2 = fminf(fmaxf(cl * kLog2e, 0x1p-100f), 0x1p80f), thr = kChGrow / c2, row_cl = cl;
      const int minpos = s.pos0 + row0 / a.hpg, maxpos = s.pos0 + (s.row0 + min(s.nrows, (i + 1) * kChM) - 1) / a.hpg;
      float m_true = -CUDART_INF_F, m_ref = -CUDART_INF_F, l = 0.f, mb = 0.f;      // mb: kProbShift less the reference
      bool far = false;                  // the row has logits beyond kFarLogit
      int id0, id1;
      pages_of(s, p0, id0, id1);
      for (int t = 0; t < n && ok; ++t) {
        const int n0 = (p0 + t) * kChN, c0 = id0, c1 = id1;
        if (t + 1 < n) pages_of(s, p0 + t + 1, id0, id1);
        ok = mbar_wait_warp(&bar->s_full[i], (sc + t) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        if (t + 1 == n) {
          ++pc;
          next = find(false);
          if (next > 0) start_q(bar->piece[pc % kChPieces]);
        }
        if (c0 < 0 || c1 < 0 || n0 + kChN - 1 > minpos || (a.window > 0 && n0 <= maxpos - a.window)) {
          int clo = a.window > 0 ? my_pos - a.window - n0 : -1, chi = my_pos - n0;       // visible columns: clo < c <= chi
          if (c0 < 0) clo = max(clo, kPageTokens - 1);
          if (c1 < 0) chi = min(chi, kPageTokens - 1);
#pragma unroll 1
          for (int c = 0; c < kChN; c += 32) {
            if (__all_sync(0xffffffffu, c > clo && c + 31 <= chi)) continue;
            uint32_t x[32];
            tmem_ld32(tS + c, x);
            tc_wait_ld();
            // bit e: column c + e is visible
            const int lo = clo + 1 - c, hi = chi - c;
            const uint32_t seen = (hi < 0 ? 0u : hi >= 31 ? 0xffffffffu : (2u << hi) - 1u) & (lo <= 0 ? 0xffffffffu : lo > 31 ? 0u : 0xffffffffu << lo);
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = seen >> e & 1 ? x[e] : 0xff800000u;
            tmem_st32(tS + c, x);
          }
          tc_wait_st();
        }
        uint32_t sv[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, sv[c]);
        tc_wait_ld();
        float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(sv[c][e]));
        m_true = fmaxf(m_true, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
        const bool first = m_ref == -CUDART_INF_F;
        const bool grow = first ? m_true > m_ref : m_true > m_ref + thr;
        const bool need_o = grow && !first;
        const float m_old = m_ref;
        if (grow) {
          m_ref = m_true;
          far = fabsf(m_ref * c2) > kFarLogit;
          mb = far ? kProbShift : kProbShift - m_ref * c2;
        }
        if (__any_sync(0xffffffffu, need_o || far)) {
          if (__any_sync(0xffffffffu, need_o)) {
            ok = mbar_wait_warp(&bar->pv_done[i], (sc + t - 1) & 1, abort);   // O_i must hold PV(t - 1) before it is scaled
            if (!ok) break;
            tc_fence_after();
            const float f = need_o ? ex2((m_old - m_ref) * c2) : 1.f;
            l *= f;
#pragma unroll 2
            for (int c = 0; c < DV / 8; ++c) {
              uint32_t ov[8];
              tmem_ld8(tO + c * 8, ov);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 8; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * f);
              tmem_st8(tO + c * 8, ov);
            }
            tc_wait_st();
          }
          if (__any_sync(0xffffffffu, far)) {
            const float m = far ? m_ref : 0.f;
#pragma unroll 1
            for (int c = 0; c < kChN; c += 32) {     // (by way of tensor memory: code that hardly ever runs stays short)
              uint32_t x[32];
              tmem_ld32(tS + c, x);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) - m);
              tmem_st32(tS + c, x);
            }
            tc_wait_st();
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, sv[c]);
            tc_wait_ld();
          }
        }
        float rs[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; c += 2) {          // probabilities take the places of the logits they come from
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int cc = c + (e >> 4), ee = (e & 15) * 2;
            const float p0 = ex2(fmaf(__uint_as_float(sv[cc][ee]), c2, mb)), p1 = ex2(fmaf(__uint_as_float(sv[cc][ee + 1]), c2, mb));
            rs[0] += p0;
            rs[1] += p1;
            sv[c][e] = h2u(__floats2half2_rn(p0, p1));
          }
          tmem_st32(tS + c * 16, sv[c]);
          if (c == 0) {
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&bar->p_half[i]);
          }
        }
        l += rs[0] + rs[1];
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(&bar->p_full[i]);
      }
      if (!ok) break;
      const int last = (sc + n - 1) & 1;
      sc += n;
      if (next > 0) finish_q();
      ok = mbar_wait_warp(&bar->pv_done[i], last, abort);
      if (!ok) break;
      tc_fence_after();
      const int row = i * kChM + r;
      const float rel = l > 0.f ? ex2((m_ref - m_true) * c2) * kProbUnshift : 1.f;       // results relative to the row's true maximum
      const float f = s.whole ? (l > 0.f ? 1.f / l : 1.f) : rel;
      float* part = s.whole ? nullptr : split_part(a, gridDim.x, kChRows, blockIdx.x, s.part);
      Segment sg;
      sg.tok0 = s.tok0; sg.row0 = s.row0; sg.g = s.g;
      const int orow = row < s.nrows ? (int)out_row(a, sg, row) : -1;
      // 64 bytes of every row of the warp at a time, through shared memory: four lanes a row on their way out instead of one
      uint8_t* stage = smem + SM::oOut + warp * 2048;
#pragma unroll 1
      for (int g = 0; g < GV; ++g) {
        uint32_t ov[32];
        tmem_ld32(tO + g * 32, ov);
        tc_wait_ld();
        if (g + 1 == GV) {
          tc_fence_before();
          mbar_arrive(&bar->o_free[i]);
        }
        // dimension 8 e + n is column 8 (n / 2) + 2 e + n % 2
        auto val = [&](int e, int n) { return __uint_as_float(ov[8 * (n >> 1) + 2 * e + (n & 1)]) * f; };
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (s.whole && half) break;
          uint4* to = reinterpret_cast<uint4*>(stage + lane * 64);
          if (s.whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              __nv_bfloat162 b[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) b[k] = __floats2bfloat162_rn(val(e, 2 * k), val(e, 2 * k + 1));
              to[e ^ (lane >> 1 & 3)] = make_uint4(*reinterpret_cast<uint32_t*>(&b[0]), *reinterpret_cast<uint32_t*>(&b[1]),
                                                   *reinterpret_cast<uint32_t*>(&b[2]), *reinterpret_cast<uint32_t*>(&b[3]));
            }
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int e = 2 * half + (q >> 1), k = 4 * (q & 1);
              to[q ^ (lane >> 1 & 3)] = make_uint4(__float_as_uint(val(e, k)), __float_as_uint(val(e, k + 1)), __float_as_uint(val(e, k + 2)), __float_as_uint(val(e, k + 3)));
            }
          }
          __syncwarp();
          const int n64 = s.whole ? g : 2 * g + half;
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const int rr = it * 8 + (lane >> 2), e = lane & 3, at = __shfl_sync(0xffffffffu, orow, rr);
            const uint4 x = *reinterpret_cast<const uint4*>(stage + rr * 64 + ((e ^ (rr >> 1 & 3)) << 4));
            uint8_t* base = s.whole ? (uint8_t*)a.out + (int64_t)at * (DV * 2) : (uint8_t*)(part + (row - lane + rr) * DV);
            if (at >= 0) *reinterpret_cast<uint4*>(base + n64 * 64 + e * 16) = x;
          }
          __syncwarp();
        }
      }
      if (row < s.nrows) {
        const float M = max_of_row(m_true == -CUDART_INF_F ? m_true : m_true * row_cl, l);
        if (s.whole) {
          a.M[orow] = M;
          a.L[orow] = logf(l * rel);
        } else {
          reinterpret_cast<float2*>(part + kChRows * DV)[row] = make_float2(M, l * rel);
        }
      }
      release(cur);
    }
  }

  // ------------------------------------------------------------ teardown (every thread gets here)
  pdl_launch();
  asm volatile("cp.async.wait_all;" ::: "memory");        // (queries that a wait which ran out left on their way)
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && bar->abort) report_timeout(timeouts);
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

static int chunk_blocks() { return 148; }

size_t cache4_chunk_workspace(const Cache4Args& a) { return split_bytes(chunk_blocks(), kChRows, a.dv); }

template <int DK, int DV>
static int launch_chunk_t(const Cache4Args& a, cudaStream_t st) {
  using SM = ChunkSmem<DK, DV>;
  auto kern = cache4_chunk_kernel<DK, DV>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::kDynamic);
  if (e != cudaSuccess) return fail(NSA_ERR_LAUNCH, "cache4_chunk: cannot reserve %d bytes of shared memory: %s", SM::kDynamic, cudaGetErrorString(e));
  // the split of registers over the roles draws on what the block is launched with
  cudaFuncAttributes at;
  e = cudaFuncGetAttributes(&at, kern);
  if (e != cudaSuccess || at.numRegs < kChRegsNeeded)
    return fail(NSA_ERR_LAUNCH, "cache4_chunk: built with %d registers a thread, the roles share %d", at.numRegs, kChRegsNeeded);
  int* timeouts = fa_timeout_counter();
  if (!timeouts) return fail(NSA_ERR_LAUNCH, "cache4_chunk: cannot set up the time-out record of this device");
  {
    KernelTimer kt("cache4_chunk", st);
    kern<<<chunk_blocks(), kChThreads, SM::kDynamic, st>>>(a, timeouts);
    if (int rc = check_launch("cache4_chunk")) return rc;
  }
  return launch_combine(a, chunk_blocks(), kChRows, false, st);
}

int launch_chunk(const Cache4Args& a, cudaStream_t st) {
  if (timeout_flagged())
    return fail(NSA_ERR_LAUNCH, "cache4_attn: a tensor-core kernel gave up on a barrier wait earlier (device time-out); results since then are "
                "invalid.  nsa_device_timeouts(1) reports and clears the condition");
  if (a.dk == 192 && a.dv == 128) return launch_chunk_t<192, 128>(a, st);
  if (a.dk == 128 && a.dv == 128) return launch_chunk_t<128, 128>(a, st);
  if (a.dk == 64 && a.dv == 64) return launch_chunk_t<64, 64>(a, st);
  return fail(NSA_ERR_UNSUPPORTED, "cache4_chunk: unsupported head dims");
}

}  // namespace nsa
