// Attention over the 4-bit latent cache, and the weights it gave every cached token.
//
// A query row r = (token t, head h) of a packed call has q_r [576]; a cached token j has the lifted latent
// c_j [512] and the roped key dims pe_j [64]. With k_j = [c_j | pe_j] and v_j = c_j:
//
//   s_rj = scale * q_r . k_j      lse_r = log sum_j exp(s_rj)      out_r = sum_j exp(s_rj - lse_r) c_j
//   weights: acc_j += sum_r exp(s_rj - lse_r)
//
// over the tokens j that row r sees: those of its sequence up to its own, or the slots it picked.
//
// Bounds. A row tile of 64 rows costs 2 * (576 + 512) * 64 = 139 kFLOP a token against the 416 bytes it
// reads: 84 ps a token at 1664 TFLOP/s, 64 ps at 6.55 TB/s. The products are turned round, S^T = K Q^T and
// O^T = C^T P^T, so that 128 tokens (then 128 latent dims) are the M of the instruction and the rows its N: 64
// heads fill it, and 16 do not pay for 64. Both read the same tile in shared memory, [token][dim], once
// K-major and once MN-major. What bounds it is shared memory, 128 bytes a clock: a tile of 128 tokens takes
// 3,090 clocks of the products' operands, 1,320 of stores, 700 of loads, 130 of barriers and 1,520 of the
// codes' way through L1, 6,750 in all of the 7,000 or so it takes (attention of 32 sequences, 64 heads: 94 us).
//
// A CTA an SM walks tiles of 128 tokens. Its eight working warps all do everything in turn, because the steps of a
// tile follow one another (one tile of lifted rows and 64 query rows fill shared memory):
//  - lift: each thread has eight 16-byte chunks of codes in registers, fetched while the tile before was
//    multiplied, lifts them (exact in f16) and stores them 128-byte swizzled, 256 dims at a time: a half is
//    refilled as soon as the products that read it are done, and the next products start on the halves there;
//  - softmax: a token a lane and 32 rows a warp, without a reduction over tokens in the common case. The
//    row's reference m is only raised, with O^T rescaled, when a score passes it by 2^8; sums stay a
//    lane's own until the end. P^T goes to shared memory as f16, in the place of the rope block.
// A ninth warp issues tcgen05.mma: S^T [128 tokens x rows] in 64 TMEM columns (f16 over the latent dims, bf16 over
// the rope dims: k_pe keeps its bf16 range), O^T [4 x 128 dims x rows] in 256.
// A call finds none of its instructions in the SMs' caches, and the steps of a tile pass through 20 KB of them, so
// the rest is kept short: with queries, raises, the rows' writing and the products unrolled, 130 KB in all for
// the 98 KB of now, the same took 111 us, and a lone short sequence 25 for 20.
// Tried: warps that only lift beside warps that only weigh (6.7 us a tile against 4.4: each idles through the
// other's half); sixteen working warps, of 104 registers (as fast; more work a tile, twice over the scores);
// pairs of 64-dim blocks a warp (10% slower: a load touches twice the lines); the codes fetched while O^T is
// multiplied (7% slower) or before the scores are read (2%).
// q goes to f16 times a power of two a row that puts its largest near 2^14: exact down to 2^-28 of it, and
// off by 2^-39 of it below. P is 2^(s - m + 7): m is at most 2^8 below the maximum, so P stays under
// 2^15, and is rounded by 2^-12 of itself down to 2^-21 of the reference (2^-32 of it below).
//
// The tiles of all (sequence, row tile) items are numbered in order and cut into equal shares, one a
// CTA: a long sequence is split over many, short ones share one. An item that a CTA holds whole is
// written out; the parts of a split one go to the workspace and glm_kv4_join adds them.
#pragma once

#include "glmkv_mqa.cuh"

namespace glmkv {

constexpr int A4_KEYS = 128, A4_ROWS = 64;
constexpr int A4_WARPS = 8;                          // working warps
// and a warpgroup of which one warp issues the products. 168 registers a thread at launch, 2016 a lane; 8 x 216
// + 4 x 64 after the split.
constexpr int A4_THREADS = 32 * (A4_WARPS + 4), A4_REGS = 216, A4_REGS_ISSUE = 64;
constexpr int A4_BLOCKS = MLA / 64;                  // 64-dim blocks: 8 latent, 1 rope
constexpr int A4_KBLK = A4_KEYS * 128;               // 16,384 B: a block of the token tile
constexpr int A4_QBLK = A4_ROWS * 128;               // 8,192 B: a block of the row tile
constexpr int A4_SMEM = 1024 + A4_BLOCKS * (A4_KBLK + A4_QBLK);  // 222,208 B with the alignment
constexpr int A4_TMEM = 512, A4_O = 0, A4_S = 256;   // O^T: four 64-column blocks; S^T: two buffers of 64
constexpr int A4_NONE = INT_MIN;
constexpr int A4_NAN = INT_MIN;                      // set in the slot of a token that has a NaN scale
constexpr float A4_LOW = -3.402823466e38f;           // a row's reference before its first token: no score is lower
constexpr float A4_OFF = 7.f, A4_TOP = 15.f;         // P = 2^(s - m + 7); m is raised past 2^15
// part of a split item: O^T as [64 rows][512] f32, then 64 references and 64 sums; two a CTA
constexpr int A4_PART = A4_ROWS * (KVL + 2) * 4;
struct A4Rec {  // the split item that starts in this CTA
  long long row0;
  int nrows, last;  // last: the CTA with its last part, -1: none
};

// kind::f16: D f32, A and B f16 (0) or bf16 (1), N >> 3 at bit 17, M = 128; bits 15, 16: MN-major A, B
__device__ __forceinline__ uint32_t a4_idesc(uint32_t type, uint32_t mn, int n) {
  return (1u << 4) | (type << 7) | (type << 10) | (mn << 15) | (mn << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// Shared-memory descriptors in the 128-byte swizzle: start address and LBO in the low word, the rest, the same
// for all, in the high one: 8-row groups 1024 bytes apart (SBO), version 1, layout 2. K-major operands do not
// use LBO. MN-major ones have 64 elements of M or N a 128-byte row, one row a k, and the next 64 elements a
// block (16,384 B) on: that is their LBO. A step adds to the low word only.
constexpr uint32_t A4_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t a4_desc(uint32_t saddr) {
  return ((saddr >> 4) & 0x3FFFu) | ((uint32_t)(A4_KBLK >> 4) << 16);
}
__device__ __forceinline__ void a4_mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(A4_DESC_HI)
      : "memory");
}
// 8 f32 columns of the warp's 32 lanes; valid on return
__device__ __forceinline__ void a4_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void a4_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ float a4_exp2(float x) {
  float d;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<const unsigned long long*>(&a)), "l"(*reinterpret_cast<const unsigned long long*>(&b)));
  return *reinterpret_cast<const float2*>(&d);
}
__device__ __forceinline__ void a4_sts(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// The working warps' barrier, and the same with an or over their 256 threads. All of them reach every one: each
// wait before it is bounded, and what they leave on is the or.
__device__ __forceinline__ void a4_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool a4_any(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v)
      : "memory");
  return r != 0;
}
// Those and the issuing warp's.
__device__ __forceinline__ void a4_all() { asm volatile("bar.sync 2, 288;" ::: "memory"); }
// The thread's number, read anew.
__device__ __forceinline__ int a4_tid() {
  int t;
  asm volatile("mov.u32 %0, %%tid.x;" : "=r"(t));
  return t;
}
// v, as a value the compiler knows nothing of: what is added to it is added where it is used, not held in a
// register from before the loop on (the descriptors of 68 products were).
__device__ __forceinline__ uint32_t a4_here(uint32_t v) {
  asm volatile("" : "+r"(v));
  return v;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r));
  return r != 0;
}

// v[k] of all 32 lanes reduced, for 32 k at once: lane l returns that of k = l. Each level halves what is left
// (31 shuffles, where 32 butterflies would take 160).
template <class Op>
__device__ __forceinline__ float a4_reduce32(float (&v)[32], int l, Op op) {
#pragma unroll
  for (int h = 16; h > 0; h >>= 1) {
    const bool up = l & h;
#pragma unroll
    for (int k = 0; k < h; ++k) {
      const float send = up ? v[k] : v[k + h], keep = up ? v[k + h] : v[k];
      v[k] = op(keep, __shfl_xor_sync(FULL, send, h));
    }
  }
  return v[0];
}

enum { A4_ATTN, A4_PICKS, A4_WEIGHTS };

struct A4Args {
  const bf16* q;
  const u8* kv;
  long long n_slots;
  const int* table;  // block table, or the picks
  int max_pages;
  const long long* cu;
  const int* lens;
  int nseq, heads, T;
  float scale;
  bf16* out;
  float* lse;
  float* acc;
  u8* ws;
};

// A run of tiles of one item: row tiles [rt0, rt1) (one, but for the weights: all the sequence's) over
// token tiles [kt0, kt1) of the item's kt.
struct A4Seg {
  int seq, rt0, rt1, kt0, kt1, kt, len, qlen;
  long long qrow;  // the sequence's first query row
  int ke;          // the tiles from here to kt1 no row sees
  int live;        // 0: no segment is left
};

// What a sequence holds, clamped to what the call's buffers do.
template <int MODE>
__device__ __forceinline__ A4Seg a4_seq(const A4Args& a, int s) {
  A4Seg g;
  g.seq = s;
  if constexpr (MODE == A4_PICKS) {
    g.len = min(max(a.lens[s], 0), TOPK), g.qlen = 1, g.qrow = (long long)s * a.heads;
  } else {
    const long long c0 = min(max(a.cu[s], 0ll), (long long)a.T), c1 = min(max(a.cu[s + 1], c0), (long long)a.T);
    // (numbers of tokens past the last tile stay ints)
    g.len = min(max(a.lens[s], 0), INT_MAX - 4 * A4_KEYS), g.qlen = (int)(c1 - c0), g.qrow = c0 * a.heads;
  }
  const long long rows = (long long)g.qlen * a.heads;
  g.rt0 = 0, g.rt1 = (int)((rows + A4_ROWS - 1) / A4_ROWS);
  g.kt0 = 0, g.kt = g.kt1 = (g.len + A4_KEYS - 1) / A4_KEYS;
  if (MODE != A4_WEIGHTS && g.kt == 0) g.kt = g.kt1 = 1;  // an empty sequence's rows are written too
  return g;
}
template <int MODE>
__device__ __forceinline__ long long a4_tiles(const A4Seg& g) {
  return MODE == A4_WEIGHTS ? (g.rt1 > 0 ? g.kt : 0) : (long long)g.rt1 * g.kt;
}
// The tokens that row r of the tile at `rt` sees: those below this.
template <int MODE>
__device__ __forceinline__ int a4_limit(const A4Args& a, const A4Seg& g, int row) {
  if constexpr (MODE == A4_PICKS) return g.len;
  return g.len - g.qlen + row / a.heads + 1;
}

// The tiles of a segment that any row sees: the rest are passed over by every role alike.
template <int MODE>
__device__ __forceinline__ int a4_kt_end(const A4Args& a, const A4Seg& g) {
  if constexpr (MODE == A4_PICKS) return min(g.kt1, (g.len + A4_KEYS - 1) / A4_KEYS);
  const long long last = min((long long)g.rt1 * A4_ROWS, (long long)g.qlen * a.heads) - 1;
  const int lim = min(g.len, max(0, a4_limit<MODE>(a, g, (int)last)));
  return min(g.kt1, (lim + A4_KEYS - 1) / A4_KEYS);
}

// The segments of this CTA's share of the tiles, in order: `left` tiles from tile kt of row tile rt of sequence
// s on (the weights: of all its row tiles).
template <int MODE>
struct A4Walk {
  long long left;
  int s, rt, kt;
  __device__ __forceinline__ void next(const A4Args& a, A4Seg& g) {
    g.live = find(a, g);
    if (g.live) g.ke = a4_kt_end<MODE>(a, g);
  }
  __device__ __forceinline__ bool find(const A4Args& a, A4Seg& g) {
    for (; left > 0 && s < a.nseq; ++s, rt = kt = 0) {
      g = a4_seq<MODE>(a, s);
      if (a4_tiles<MODE>(g) == 0 || rt >= g.rt1) continue;
      g.kt0 = kt, g.kt1 = (int)min((long long)g.kt, kt + left);
      left -= g.kt1 - g.kt0;
      if constexpr (MODE == A4_WEIGHTS) {
        rt = g.rt1;  // the next call goes on to the next sequence
      } else {
        g.rt0 = rt, g.rt1 = rt + 1;
        ++rt, kt = 0;
      }
      return true;
    }
    return false;
  }
};

// What a thread lifts of a tile: one 16-byte chunk of its half's codes, with its two scales, of eight tokens.
struct A4Raw {
  uint4 nib[2][4];
  uint32_t sc[2][4];
};

template <int MODE>
__device__ __forceinline__ void a4_run(const A4Args& a) {
  extern __shared__ __align__(1024) u8 a4_raw[];
  __shared__ __align__(8) unsigned long long k_full[3], k_free[3], q_full, s_full[2], p_full, mma_done;
  __shared__ __align__(16) float cf[4][A4_ROWS];   // a row's score factor, scale / its power of two; a ring
  __shared__ __align__(16) float nm[A4_ROWS];      // minus its reference (weights: minus its lse)
  __shared__ __align__(16) float fac[A4_ROWS];
  __shared__ float wred[4][A4_ROWS];
  __shared__ float wpart[2][A4_KEYS];              // weights: the sums of the warps that do not add them
  __shared__ int lim[A4_ROWS];
  __shared__ int slots[4][A4_KEYS];                // each token's slot, -1: not there, A4_NAN set: NaN; a ring
  __shared__ A4Walk<MODE> walk_s;
  __shared__ A4Seg segs[2];                        // the segment at work, and the one after it
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  __shared__ long long w_share;                    // a CTA's tiles, and how many CTAs have one more
  __shared__ int w_rest;
  const int tid = threadIdx.x, warp = __shfl_sync(FULL, tid >> 5, 0), l = tid & 31;
  const uint32_t kbuf = (smem_u32(a4_raw) + 1023u) & ~1023u, qbuf = kbuf + A4_BLOCKS * A4_KBLK;
  const uint32_t pbuf = kbuf + 8 * A4_KBLK;  // P^T [token][row] takes the rope block's place
  constexpr float LOG2E = 1.4426950408889634f;
  if (tid == 0) {
    // the two halves of the latent blocks, and the rope block
    for (int i = 0; i < 3; ++i) mbar_init(smem_u32(&k_full[i]), A4_WARPS), mbar_init(smem_u32(&k_free[i]), 1);
    mbar_init(smem_u32(&q_full), A4_WARPS);
    mbar_init(smem_u32(&s_full[0]), 1);
    mbar_init(smem_u32(&s_full[1]), 1);
    mbar_init(smem_u32(&p_full), A4_WARPS);
    mbar_init(smem_u32(&mma_done), 1);
    mbar_init_fence();
    abort_flag = 0;
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "r"(A4_TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  pdl_trigger();  // one CTA an SM, all resident
  pdl_wait();
  // ---- this CTA's share of the tiles. Thread i counts the sequences [i c, (i + 1) c); the warps' counts go where
  // the tiles go later.
  long long* const counts = reinterpret_cast<long long*>(a4_raw);
  const int c = (a.nseq + A4_THREADS - 1) / A4_THREADS, s0 = min(a.nseq, tid * c), s1 = min(a.nseq, s0 + c);
  long long mine = 0;
  for (int s = s0; s < s1; ++s) mine += a4_tiles<MODE>(a4_seq<MODE>(a, s));
  long long before = mine, total = 0;  // the tiles of the sequences before this thread's; all
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(FULL, before, o);
    if (l >= o) before += y;
  }
  if (l == 31) counts[warp] = before;
  if (tid == 0) walk_s.left = 0;
  __syncthreads();
  tc_fence_after();
  before -= mine;
#pragma unroll
  for (int w = 0; w < A4_THREADS / 32; ++w) {
    const long long n = counts[w];
    if (w < warp) before += n;
    total += n;
  }
  // a CTA's tiles, and how many CTAs have one more
  const bool small = total <= INT_MAX;
  const long long share = small ? (int)total / (int)gridDim.x : total / gridDim.x;
  const int rest = (int)(total - share * gridDim.x);
  if (tid == 0) w_share = share, w_rest = rest;
  const long long t0 = blockIdx.x * share + min((int)blockIdx.x, rest), t1 = t0 + share + ((int)blockIdx.x < rest);
  if (before <= t0 && t0 < before + mine) {  // one thread, if t0 < total: its sequences hold tile t0
    long long base = before;
    int s = s0;
    for (; s < s1; ++s) {
      const long long n = a4_tiles<MODE>(a4_seq<MODE>(a, s));
      if (t0 < base + n) break;
      base += n;
    }
    A4Walk<MODE> w{t1 - t0, s, 0, (int)(t0 - base)};
    if (MODE != A4_WEIGHTS) {
      const int kt = a4_seq<MODE>(a, s).kt;
      w.rt = (int)((t0 - base) / kt), w.kt = (int)((t0 - base) % kt);
    }
    walk_s = w;
  }
  __syncthreads();
  auto first_tile = [&](int b) { return b * w_share + min(b, w_rest); };
  const uint32_t tmem = tmem_base;
  const volatile int* abort = &abort_flag;
  auto give_up = [&]() {
    atomicOr(&g_fault, FAULT_WAIT_TIMEOUT);
    abort_flag = 1;
  };
  if (warp >= A4_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(A4_REGS_ISSUE));
    if (warp > A4_WARPS) {
      __syncthreads();  // with the one at the end
      return;
    }
    // ---------------------------------------------------------------- the products, by one lane of this warp
    // All its lanes walk and wait together, and the lane is elected: the descriptors then stay in uniform
    // registers. One lane branching off alone took 55 to 65 clocks a product where the hardware takes 48.
    const bool lane = elect_one();
    const uint32_t kd0 = a4_desc(kbuf), qd0 = a4_desc(qbuf);
    uint32_t tile = 0, step = 0, item = 0;
    bool ok = true, issued = false;
    A4Walk<MODE> walk = walk_s;
    __syncwarp();
    a4_all();  // before the working warps step theirs
    A4Seg g;
    for (walk.next(a, g); g.live && ok; walk.next(a, g)) {
      const int ke = g.ke, nrt = MODE == A4_WEIGHTS ? g.rt1 - g.rt0 : 1;
      for (int kt = g.kt0; kt < ke && ok; ++kt) {
        for (int rt = g.rt0; rt < g.rt0 + nrt && ok; ++rt) {
          const int nrows = (int)min((long long)A4_ROWS, (long long)g.qlen * a.heads - (long long)rt * A4_ROWS);
          const int n = (nrows + 15) & ~15;
          if (kt == g.kt0 || nrt > 1) ok = mq_wait(smem_u32(&q_full), item++ & 1, abort);
          const uint32_t d = tmem + A4_S + 64 * (step & 1);
          const bool lastk = rt == g.rt0 + nrt - 1;
#pragma unroll
          for (int p = 0; p < 3; ++p) {  // each half, and the rope block, as it is there
            if (rt == g.rt0) ok = ok && mq_wait(smem_u32(&k_full[p]), tile & 1, abort);
            ok = __all_sync(FULL, ok);
            if (!ok) break;
            // The stores that the barriers tell of, made visible to the tensor cores' reads. By this warp: the
            // writers' own fences would wait for their loads, a memory latency each.
            fence_async_smem();
            tc_fence_after();
            if (lane) {
              const uint32_t id = a4_idesc(p < 2 ? 0u : 1u, 0u, n), kd = a4_here(kd0), qd = a4_here(qd0);
#pragma unroll 1
              for (int b = 4 * p; b < min(4 * p + 4, A4_BLOCKS); ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  a4_mma(d, kd + b * (A4_KBLK >> 4) + 2 * k, qd + b * (A4_QBLK >> 4) + 2 * k, id, b > 0 || k > 0);
              if (p == 2) tc_commit(smem_u32(&s_full[step & 1]));
            }
            issued = true;
          }
          if (!ok) break;
          ++step;
          if (MODE != A4_WEIGHTS) {  // O^T += C^T P^T
            ok = __all_sync(FULL, mq_wait(smem_u32(&p_full), tile & 1, abort));
            if (!ok) break;
            fence_async_smem();
            tc_fence_after();
            if (lane) {
              const uint32_t id = a4_idesc(0u, 1u, n), kd = a4_here(kd0);
#pragma unroll 1
              for (int m = 0; m < 4; ++m) {
#pragma unroll
                for (int k = 0; k < A4_KEYS / 16; ++k)
                  a4_mma(tmem + A4_O + 64 * m, kd + 2 * m * (A4_KBLK >> 4) + 128 * k, kd + 8 * (A4_KBLK >> 4) + 128 * k,
                         id, kt > g.kt0 || k > 0);
                if (m == 1) tc_commit(smem_u32(&k_free[0]));
              }
              tc_commit(smem_u32(&k_free[1]));
              tc_commit(smem_u32(&k_free[2]));  // all of the tile's products
            }
          }
          if (lastk) ++tile;
        }
      }
    }
    if (!ok && l == 0) give_up();
    if (issued) {  // every product is done before TMEM is freed
      if (lane) tc_commit(smem_u32(&mma_done));
      mbar_wait_bounded(smem_u32(&mma_done), 0, WAIT_LIMIT_NS);
    }
    tc_fence_before();
    __syncthreads();  // with the one at the end
    return;
  }
  // ---------------------------------------------------------------- the working warps
  // The walk and its segments live in shared memory, stepped by one thread: they would take 30 registers.
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(A4_REGS));
  bool ok = true;  // this warp's waits came through
  a4_all();  // the issuing warp has its walk
  // One thread steps the walk, and sends for the new segment's queries.
  auto step_walk = [&](A4Seg& s) {
    A4Walk<MODE> walk = walk_s;
    walk.next(a, s);
    walk_s = walk;
    if (s.live) {
      const long long n = min((long long)A4_ROWS, (long long)s.qlen * a.heads - (long long)s.rt0 * A4_ROWS);
      prefetch_l2(a.q + (s.qrow + (long long)s.rt0 * A4_ROWS) * MLA, (uint32_t)n * (2 * MLA));
    }
  };
  if (tid == 0) step_walk(segs[0]);
  // lift: chunk `c8` of a half's eight 16-byte chunks a row, tokens t4 + 4 i, one half after the other (a load of
  // the warp touches 4 rows of 128 bytes: it takes a cycle a line, and eight rows of 64 bytes took 16); k_pe:
  // chunk l % 8 of tokens 16 warp + l / 8 + 4 h; softmax: token `tok`, rows r0 .. r0 + 31. Each is worked out from
  // the thread's number where it is used: held all along, they cost the registers of the fetched codes. The
  // slots of a tile's tokens (token tid's by thread tid) are put down two tiles ahead, from a table entry
  // loaded a tile before that.
  uint32_t tile = 0, step = 0, item = 0;  // token tiles lifted, products of scores issued, query tiles loaded

  // Token tid of tile kt of a segment: its table entry (or pick), -1 past the table, A4_NONE past the
  // segment's tokens; and that entry's slot, or -1.
  auto entry_of = [&](const A4Seg& g, int kt) -> int {
    const int k = kt * A4_KEYS + tid;
    if (kt >= g.ke || k >= g.len) return A4_NONE;
    if constexpr (MODE == A4_PICKS) return a.table[(size_t)g.seq * TOPK + k];
    return k / PAGE < a.max_pages ? a.table[(size_t)g.seq * a.max_pages + k / PAGE] : -1;
  };
  auto slot_of = [&](int entry) -> int {
    if (entry == A4_NONE || (MODE == A4_PICKS && entry < 0)) return -1;
    const long long s = MODE == A4_PICKS ? entry : (long long)entry * PAGE + (tid & (PAGE - 1));
    if (s < 0 || s >= a.n_slots) {
      atomicOr(&g_fault, MODE == A4_PICKS ? FAULT_BAD_PICK : FAULT_BAD_PAGE);
      return -1;
    }
    return (int)s;
  };
  auto put_slot = [&](uint32_t tl, int entry) {
    const int s = slot_of(entry);
    slots[tl & 3][tid] = s;
    // the rest of the token's page, sent for to L2 by its first thread. (A prefetch a row, by 128 threads,
    // took their four warps 3,000 clocks a tile; picked rows go without.)
    if (MODE != A4_PICKS && (tid & (PAGE - 1)) == 0 && s >= 0) prefetch_l2(a.kv + (size_t)s * KV4, KV4_PAGE);
  };
  int nent = A4_NONE;  // threads below 128: the entry of the tile three ahead
  A4Raw raw;
  // The codes of tile tl, one half after the other. A token that is not there reads slot 0, with scales of zero.
  auto fetch = [&](uint32_t tl) {
    const int th = a4_tid(), c8 = (th & 31) >> 2, t4 = 16 * (th >> 5) + (th & 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = slots[tl & 3][t4 + 4 * i];
      const u8* src = a.kv + (size_t)max(s, 0) * KV4;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        raw.nib[h][i] = __ldg(reinterpret_cast<const uint4*>(src + 16 * c8) + 8 * h);
        raw.sc[h][i] = s < 0 ? 0u : __ldg(reinterpret_cast<const uint16_t*>(src + KV4_SC + 2 * c8) + 8 * h);
      }
    }
  };

  // Row tile rt's queries. The scores of those before are done: every warp has waited for them.
  auto queries = [&](const A4Seg& g, int rt) {
    const int th = a4_tid(), l = th & 31, warp = th >> 5;
    const int nrows = (int)min((long long)A4_ROWS, (long long)g.qlen * a.heads - (long long)rt * A4_ROWS);
    const uint4* src = reinterpret_cast<const uint4*>(a.q + (g.qrow + (long long)rt * A4_ROWS) * MLA) + l;
    uint4 nx[2][3];
    auto load = [&](int r) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 3; ++k)
          nx[i][k] = r + i < nrows && (k < 2 || l < 8) ? __ldg(src + (r + i) * (MLA / 8) + 32 * k) : make_uint4(0, 0, 0, 0);
    };
    load(warp * 8);
    // Two rows at a time: all eight at once were 30 KB of instructions, fetched anew by every call.
#pragma unroll 1
    for (int r = warp * 8; r < warp * 8 + 8; r += 2) {
      uint4 v[2][3];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 3; ++k) v[i][k] = nx[i][k];
      if (r < warp * 8 + 6) load(r + 2);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t mx = 0;
#pragma unroll
        for (int k = 0; k < 3; ++k)
          mx = absmax_xs(mx, absmax_xs(absmax_xs(v[i][k].x, v[i][k].y), absmax_xs(v[i][k].z, v[i][k].w)));
        const float top = warp_max(absmax_bf16x2(mx));
        const int e = (int)(__float_as_uint(top) >> 23);
        // the row's power of two: its largest to [2^14, 2^15) (all zeros, inf: as it is)
        const int fe = e == 0 || e == 255 ? 127 : min(268 - e, 253);
        const float f = __uint_as_float((uint32_t)fe << 23), inv = __uint_as_float((uint32_t)(254 - fe) << 23);
        if (l == 0) cf[item & 3][r + i] = a.scale * inv * (MODE == A4_WEIGHTS ? 1.f : LOG2E);
#pragma unroll
        for (int k = 0; k < 3; ++k) {  // 16-byte chunk 32 k + l of the row, in 64-dim block 4 k + l / 8
          const uint32_t w[4] = {v[i][k].x, v[i][k].y, v[i][k].z, v[i][k].w};
          uint32_t o[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float2 y = mul2(unpack2(w[x]), make_float2(f, f));
            if (k < 2) {
              const __half2 hh = __floats2half2_rn(y.x, y.y);
              o[x] = *reinterpret_cast<const uint32_t*>(&hh);
            } else {
              o[x] = pack_bf16x2(y.x, y.y);
            }
          }
          if (k < 2 || l < 8)
            a4_sts(qbuf + (4 * k + (l >> 3)) * A4_QBLK + (r + i) * 128 + (((l & 7) ^ ((r + i) & 7)) << 4),
                   make_uint4(o[0], o[1], o[2], o[3]));
        }
      }
    }
    tc_fence_before();  // this warp's reads of the scores two steps ago
    __syncwarp();
    if (l == 0) mbar_arrive(smem_u32(&q_full));
    ++item;
  };
  // What the next scores need: row tile rt's queries where they change, the tile in `raw` where it does.
  // `more`: a tile follows in the segment; `after()`: for threads below 128, their entry of the tile three on.
  auto prepare = [&](const A4Seg& g, int rt, bool newq, bool newk, bool more, auto&& after) {
    if (newq) queries(g, rt);
    if (newk) {
      tc_fence_before();  // as above
      const int th = a4_tid(), l = th & 31, warp = th >> 5, c8 = l >> 2, t4 = 16 * warp + (l & 3);
      // k_pe goes as it is, loaded now for the end
      const int key = 16 * warp + (l >> 3);
      uint4 pe[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int ks = slots[tile & 3][key + 4 * h];
        pe[h] = ks < 0 ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(a.kv + (size_t)ks * KV4 + KV4_PE) + (l & 7));
      }
      if constexpr (MODE == A4_ATTN) {
        // A NaN scale (the append gives a group one that has a NaN latent) would reach rows that do not see the token, as
        // 0 * NaN: it is lifted as zeros, and the token's scores are made NaN instead.
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) bad |= (raw.sc[i / 4][i % 4] & 0x7f7fu) + 0x0101u;
        if (bad & 0x8080u) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (((raw.sc[i / 4][i % 4] & 0x7f7fu) + 0x0101u) & 0x8080u) {
              raw.sc[i / 4][i % 4] = 0;
              slots[tile & 3][t4 + 4 * (i % 4)] |= A4_NAN;  // (this warp's tokens alone; the scores' barriers tell of it)
            }
        }
      }
      ++tile;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // the products of the tile before have read this half (the weights: their scores are there already)
        if (MODE != A4_WEIGHTS && tile > 1 && ok) ok = mq_wait(smem_u32(&k_free[h]), tile & 1, abort);
        const uint32_t dst = kbuf + (4 * h + (c8 >> 1)) * A4_KBLK, c0 = (c8 & 1) << 6;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // (t4 + 4 i) % 8 = l % 4 + 4 (i % 2)
          const uint32_t row = dst + (t4 + 4 * i) * 128, sr = ((l & 3) << 4) | ((i & 1) << 6);
          __half2 sc0, sc1;
          kv4_scales((uint16_t)raw.sc[h][i], sc0, sc1);
          a4_sts(row + ((c0 + 0) ^ sr), kv4_lift8(raw.nib[h][i].x, sc0));
          a4_sts(row + ((c0 + 16) ^ sr), kv4_lift8(raw.nib[h][i].y, sc0));
          a4_sts(row + ((c0 + 32) ^ sr), kv4_lift8(raw.nib[h][i].z, sc1));
          a4_sts(row + ((c0 + 48) ^ sr), kv4_lift8(raw.nib[h][i].w, sc1));
        }
        __syncwarp();
        if (l == 0) mbar_arrive(smem_u32(&k_full[h]));
      }
      if (MODE != A4_WEIGHTS && tile > 1 && ok) ok = mq_wait(smem_u32(&k_free[2]), tile & 1, abort);
      const uint32_t row = kbuf + 8 * A4_KBLK + key * 128;  // (a token's place in its eight: l >> 3, and 4 more)
#pragma unroll
      for (int h = 0; h < 4; ++h) a4_sts(row + 512 * h + (((l & 7) ^ ((l >> 3) + 4 * (h & 1))) << 4), pe[h]);
      __syncwarp();
      if (l == 0) mbar_arrive(smem_u32(&k_full[2]));
      // the slots (they would hold up the lift, and behind the next tile's loads they wait for those: 2%), and
      // the next tile's codes, while this one's products run
      if (tid < A4_KEYS) {
        put_slot(tile + 1, nent);
        nent = after();
      }
      if (more) fetch(tile);
    }
    ++step;
  };

  if (MODE != A4_WEIGHTS && tid == 0) reinterpret_cast<A4Rec*>(a.ws)[blockIdx.x].last = -1;
  // A segment's first tile: its queries, the slots of its first tiles and its codes on their way. This is done
  // while the segment before has its last products to come, so that the new scores are worked out while its
  // rows are written.
  auto begin = [&](const A4Seg& s) {
    int e0 = A4_NONE, e1 = A4_NONE;
    if (tid < A4_KEYS) e0 = entry_of(s, s.kt0), e1 = entry_of(s, s.kt0 + 1), nent = entry_of(s, s.kt0 + 2);
    queries(s, s.rt0);
    if (tid < A4_KEYS) put_slot(tile, e0), put_slot(tile + 1, e1);
    a4_sync();
    fetch(tile);
  };
  a4_sync();
  bool ready = false;  // the segment's first tile has been prepared
  for (int at = 0; segs[at].live; at ^= 1) {
    const A4Seg &g = segs[at], &gn = segs[at ^ 1];
    a4_sync();  // the segment before has been worked with: its place, lim and nm are free
    const int nrt = MODE == A4_WEIGHTS ? g.rt1 - g.rt0 : 1;
    auto references = [&](int rt) {  // a row tile's limits and references
      const int nrows = (int)min((long long)A4_ROWS, (long long)g.qlen * a.heads - (long long)rt * A4_ROWS);
      if (tid < A4_ROWS) {
        const bool live = tid < nrows;
        lim[tid] = live ? a4_limit<MODE>(a, g, rt * A4_ROWS + tid) : 0;
        if constexpr (MODE == A4_WEIGHTS) {
          const float v = live ? a.lse[g.qrow + (long long)rt * A4_ROWS + tid] : -INFINITY;
          nm[tid] = v == -INFINITY ? v : -v;  // an empty row weighs nothing
        } else {
          nm[tid] = live ? -A4_LOW : -INFINITY;  // rows past the tile's weigh nothing
        }
      }
    };
    const int ke = g.ke;
    const bool any = g.kt0 < ke;
    references(g.rt0);
    a4_sync();
    // The segment after this, for all to read past the next barrier: in a first tile's raise, in begin(), or, for the
    // weights of a tile prepared before, the one after the wait for its scores, which the walk is stepped under.
    if (tid == 0) step_walk(segs[at ^ 1]);
    [[maybe_unused]] float sum[32];
    if constexpr (MODE != A4_WEIGHTS) {
#pragma unroll
      for (int i = 0; i < 32; ++i) sum[i] = 0.f;
    }
    int nrows = (int)min((long long)A4_ROWS, (long long)g.qlen * a.heads - (long long)g.rt0 * A4_ROWS);
    // Steps: (token tile, row tile) in order, from one before the first, which only gets that one ready, where
    // the segment before has not.
    [[maybe_unused]] float wsum = 0.f;
    int kt = any ? g.kt0 : ke, rt = ready ? g.rt0 : g.rt0 - 1;
    ready = false;
    while (kt < ke) {
      const bool first = rt < g.rt0, wrap = !first && rt + 1 == g.rt0 + nrt;
      const int kt2 = wrap ? kt + 1 : kt, rt2 = wrap ? g.rt0 : rt + 1;  // the next step
      const int th = a4_tid(), l = th & 31, warp = th >> 5, tok = th & 127, r0 = 32 * (th >> 7), sw = (th & 7) << 4;
      const uint32_t lanes = tmem + ((uint32_t)(th & 96) << 16);
      const uint32_t sbuf = (step - 1) & 1;
      const uint32_t ts = lanes + A4_S + 64 * sbuf + r0;
      const float* f = cf[(item - 1) & 3] + r0;
      const int k = kt * A4_KEYS + tok;
      int slot = -1;
      bool masked = true;  // whether a row of the tile may not see this token
      if (!first) {
        ok = __all_sync(FULL, ok && mq_wait(smem_u32(&s_full[sbuf]), ((step - 1) >> 1) & 1, abort));
        tc_fence_after();
        if (ok) slot = slots[(tile - 1) & 3][tok];
        if constexpr (MODE == A4_WEIGHTS) {
          if (nrt > 1) {
            if (a4_any(!ok)) goto out;  // and the step before is done with the references
            nrows = (int)min((long long)A4_ROWS, (long long)g.qlen * a.heads - (long long)rt * A4_ROWS);
            if (kt > g.kt0 || rt > g.rt0) {
              references(rt);
              a4_sync();
            }
          } else if (kt == g.kt0) {
            a4_sync();  // the segment after this is read below, and a tile of one row tile has no barrier before that
          }
        }
        masked = slot < 0 || k >= lim[0];
      }
      if constexpr (MODE != A4_WEIGHTS) {
        if (!first) {
          // p = 2^x, x = s - m + 7 in powers of two, of this token and its 32 rows, 0 where not seen; and P^T
          // [token][row] in f16 over the rope block, which the scores' products have read. The largest x.
          float p[32];
          auto weigh = [&]() {
            float mx = -INFINITY;
            // -0, which the compiler does not know (heads <= 1024): a product as an fma with it. A packed multiply
            // with a packed add behind it comes out fused (one rounding, measured), although both say .rn.
            const float z = __uint_as_float(0x80000000u + ((uint32_t)a.heads >> 11));
            const float2 mz = make_float2(z, z);
#pragma unroll
            for (int j = 0; j < 32; j += 16) {
              if (r0 + j >= nrows) {
#pragma unroll
                for (int i = 0; i < 16; ++i) p[j + i] = 0.f;
                break;
              }
              uint32_t u[16];
              tc_ld16_issue(ts + j, u);
              tc_ld16_wait(u);
              float* x = p + j;
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const float4 f4 = *reinterpret_cast<const float4*>(f + j + i);
                const float4 n4 = *reinterpret_cast<const float4*>(nm + r0 + j + i);
                // The score is rounded before the reference is taken off, as in the maximum that set it: past 2^28
                // that rounding is more than a weight's exponent has room for, and a fused difference would show it.
                const float2 lo = add2(fma2(make_float2(__uint_as_float(u[i]), __uint_as_float(u[i + 1])),
                                            make_float2(f4.x, f4.y), mz), make_float2(n4.x, n4.y));
                const float2 hi = add2(fma2(make_float2(__uint_as_float(u[i + 2]), __uint_as_float(u[i + 3])),
                                            make_float2(f4.z, f4.w), mz), make_float2(n4.z, n4.w));
                x[i] = lo.x, x[i + 1] = lo.y, x[i + 2] = hi.x, x[i + 3] = hi.y;
              }
              if (masked) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  if (slot == -1 || k >= lim[r0 + j + i]) x[i] = -INFINITY;
                  else if (slot < 0) x[i] = __int_as_float(0x7fffffff);
              }
              uint32_t o[8];
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                mx = fmaxf(mx, fmaxf(x[i], x[i + 1]));
                x[i] = a4_exp2(x[i]), x[i + 1] = a4_exp2(x[i + 1]);
                const __half2 h = __floats2half2_rn(x[i], x[i + 1]);
                o[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
              }
              a4_sts(pbuf + tok * 128 + ((2 * r0 + 2 * j) ^ sw), make_uint4(o[0], o[1], o[2], o[3]));
              a4_sts(pbuf + tok * 128 + ((2 * r0 + 2 * j + 16) ^ sw), make_uint4(o[4], o[5], o[6], o[7]));
            }
            return mx;
          };
          const bool work = ok && r0 < nrows;
          bool raise = kt == g.kt0;  // the first tile's references are its own
#pragma unroll 1
          for (int pass = 0;; ++pass) {
            if (!raise) {
              float mx = -INFINITY;
              if (work) mx = weigh();
              raise = a4_any(!ok || mx > A4_TOP);
              if (!raise || pass > 0) break;
            }
            if (a4_any(!ok)) goto out;
            raise = false;
            // ---- raise the references to the tile's maxima, and bring sums and O^T to them
            if (work) {
#pragma unroll
              for (int j = 0; j < 32; j += 16) {
                uint32_t u[16];  // (rows past the tile's have maxima that nothing reads)
                tc_ld16_issue(ts + j, u);
                tc_ld16_wait(u);
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                  const float4 f4 = *reinterpret_cast<const float4*>(f + j + i);
                  p[j + i] = __uint_as_float(u[i]) * f4.x, p[j + i + 1] = __uint_as_float(u[i + 1]) * f4.y;
                  p[j + i + 2] = __uint_as_float(u[i + 2]) * f4.z, p[j + i + 3] = __uint_as_float(u[i + 3]) * f4.w;
                }
                if (masked) {
#pragma unroll
                  for (int i = 0; i < 16; ++i)
                    if (slot < 0 || k >= lim[r0 + j + i]) p[j + i] = -INFINITY;
                }
              }
              wred[warp & 3][r0 + l] = a4_reduce32(p, l, [](float p, float q) { return fmaxf(p, q); });
            }
            a4_sync();
            if (tid < nrows) {
              const float v = fmaxf(fmaxf(wred[0][tid], wred[1][tid]), fmaxf(wred[2][tid], wred[3][tid])) - A4_OFF;
              const float old = -nm[tid], m = fmaxf(old, v);
              fac[tid] = a4_exp2(old - m);
              nm[tid] = -m;
            }
            a4_sync();
            // (the products of the tile before are done: every warp has waited for them)
            if (kt > g.kt0 && work) {
#pragma unroll
              for (int i = 0; i < 32; ++i) sum[i] *= r0 + i < nrows ? fac[r0 + i] : 0.f;
#pragma unroll 1
              for (int m = 0; m < 16; ++m) {
                if (r0 + 8 * (m & 3) >= nrows) continue;
                const uint32_t to = lanes + A4_O + 64 * (m >> 2) + r0 + 8 * (m & 3);
                const float* fc = fac + r0 + 8 * (m & 3);
                uint32_t u[8];
                a4_ld8(to, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * fc[i]);
                a4_st8(to, u);
              }
              asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
          }
          tc_fence_before();
          __syncwarp();
          if (l == 0) mbar_arrive(smem_u32(&p_full));
          if (work) {
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[i] += p[i];
          }
        }
      }
      // the next step, which may be the next segment's first
      const bool over = !first && kt2 >= ke && gn.live && gn.kt0 < gn.ke, start = first || over;
      const A4Seg& s2 = over ? gn : g;
      if (start) begin(s2);
      if (kt2 < ke || over) {
        const int k2 = over ? s2.kt0 : kt2;
        prepare(s2, rt2, !start && nrt > 1, first || wrap, k2 + 1 < s2.ke, [&]() -> int {
          // token tid's entry of the tile three on; past the last one of the next segment's, to send for them
          if (tid >= A4_KEYS) return A4_NONE;
          if (start || k2 + 3 < ke) return entry_of(s2, k2 + 3);
          return gn.live ? entry_of(gn, gn.kt0 + (k2 + 3 - ke)) : A4_NONE;
        });
        ready = over;
      }
      if constexpr (MODE == A4_WEIGHTS) {  // while the next step's products run, into the other buffer
        if (!first) {
#pragma unroll
          for (int j = 0; j < 32; j += 16) {
            if (r0 + j >= nrows) break;
            uint32_t u[16];
            tc_ld16_issue(ts + j, u);
            float2 nr[8], d[8];
            float low = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              const float4 n4 = *reinterpret_cast<const float4*>(nm + r0 + j + 2 * i);
              nr[i] = make_float2(n4.x, n4.y), nr[i + 1] = make_float2(n4.z, n4.w);
              low = fminf(low, fminf(fminf(n4.x, n4.y), fminf(n4.z, n4.w)));
            }
            tc_ld16_wait(u);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              // the difference in natural units first: its rounding is relative to what is left
              const float4 f4 = *reinterpret_cast<const float4*>(f + j + 2 * i);
              d[i] = fma2(make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])), make_float2(f4.x, f4.y), nr[i]);
              d[i + 1] = fma2(make_float2(__uint_as_float(u[2 * i + 2]), __uint_as_float(u[2 * i + 3])),
                              make_float2(f4.z, f4.w), nr[i + 1]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              d[i] = mul2(d[i], make_float2(LOG2E, LOG2E));
              d[i].x = a4_exp2(d[i].x), d[i].y = a4_exp2(d[i].y);
            }
            if (masked || low == -INFINITY) {  // rows that do not see this token, and empty ones
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                if (slot < 0 || k >= lim[r0 + j + 2 * i] || nr[i].x == -INFINITY) d[i].x = 0.f;
                if (slot < 0 || k >= lim[r0 + j + 2 * i + 1] || nr[i].y == -INFINITY) d[i].y = 0.f;
              }
            }
#pragma unroll
            for (int i = 1; i < 8; ++i) d[0] = add2(d[0], d[i]);
            wsum += d[0].x + d[0].y;
          }
          if (wrap) {
            // one add a token, rows summed in the same order every time: the same result, unless
            // sequences of the call share the page
            float* wp = wpart[kt & 1];
            if (r0 > 0) wp[tok] = wsum;
            if (a4_any(!ok)) goto out;
            if (r0 == 0 && slot >= 0) atomicAdd(a.acc + slot, wsum + wp[tok]);
            wsum = 0.f;
          }
        }
      }
      kt = kt2, rt = rt2;
    }
    if constexpr (MODE != A4_WEIGHTS) {
      // ---- the segment's rows: O^T over the sums, or a part of them
      const int th = a4_tid(), l = th & 31, warp = th >> 5, tok = th & 127, r0 = 32 * (th >> 7);
      const uint32_t lanes = tmem + ((uint32_t)(th & 96) << 16);
      const bool whole = g.kt0 == 0 && g.kt1 == g.kt;
      if (any) {
        // the last products (waited for already where the next segment's tile has taken the place)
        if (!ready) ok = ok && mq_wait(smem_u32(&k_free[2]), (tile - 1) & 1, abort);
        if (a4_any(!ok)) goto out;
        tc_fence_after();
      }
      const float t32 = a4_reduce32(sum, l, [](float p, float q) { return p + q; });
      wred[warp & 3][r0 + l] = t32;
      a4_sync();
      const long long row0 = g.qrow + (long long)g.rt0 * A4_ROWS;
      const int slot = g.kt0 > 0 ? 2 * blockIdx.x : 2 * blockIdx.x + 1;  // continues an item, or starts one
      u8* pt = a.ws + (size_t)gridDim.x * sizeof(A4Rec) + (size_t)slot * A4_PART;
      if (tid < A4_ROWS) {
        const float t = (wred[0][tid] + wred[1][tid]) + (wred[2][tid] + wred[3][tid]), m = -nm[tid];
        fac[tid] = whole ? (t > 0.f ? __fdividef(1.f, t) : (t == 0.f ? 0.f : t)) : 1.f;
        if (whole) {
          if (tid < nrows) a.lse[row0 + tid] = t == 0.f ? -INFINITY : (m + log2f(t)) * 0.6931471805599453f;
        } else {
          float* st = reinterpret_cast<float*>(pt) + A4_ROWS * KVL;
          st[tid] = m, st[A4_ROWS + tid] = t;
        }
      }
      if (tid == 0 && g.kt0 == 0 && !whole) {
        long long end = g.kt - g.kt1;  // the tiles left to the CTAs after this one
        int b = blockIdx.x;
        while (end > 0) ++b, end -= first_tile(b + 1) - first_tile(b);
        A4Rec rec;
        rec.row0 = row0, rec.nrows = nrows, rec.last = b;
        reinterpret_cast<A4Rec*>(a.ws)[blockIdx.x] = rec;
      }
      a4_sync();
      if (r0 < nrows) {
        bf16* const out = a.out + (row0 + r0) * KVL + tok;
        float* const po = reinterpret_cast<float*>(pt) + r0 * KVL + tok;
#pragma unroll 1
        for (int m = 0; m < KVL; m += 128) {  // dims m + tok
          uint32_t u[2][16];
          tc_ld16_issue(lanes + A4_O + m / 2 + r0, u[0]);
          tc_ld16_issue(lanes + A4_O + m / 2 + r0 + 16, u[1]);
          tc_ld16_wait(u[0]);
          tc_ld16_after(u[1]);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (r0 + i >= nrows) break;
            const float v = any ? __uint_as_float(u[i / 16][i % 16]) * fac[r0 + i] : 0.f;
            if (whole) out[m + i * KVL] = __float2bfloat16_rn(v);
            else po[m + i * KVL] = v;
          }
        }
      }
      tc_fence_before();  // read before the next segment's first product into it (it waits for p_full)
    }
  }
out:
  if (!ok && l == 0) give_up();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(A4_TMEM) : "memory");
  }
}

constexpr int J4_WARPS = 16, J4_THREADS = 32 * J4_WARPS, J4_MAX = 512;  // a CTA's; SMs at most

// The rows of the split items: each one's parts brought to their largest reference and added, in a fixed
// order. A row is bound by the latency of its parts (2 KB each, from L2), so it gets a warp, four or all 16 of
// a CTA by how many there are; each takes every 1st, 4th or 16th part, 16 dims a lane, and they are added
// through shared memory. (Groups of 128 threads with a row after another took 35 us for 4,096 rows of three
// parts.)
__device__ __forceinline__ void a4_join(const u8* __restrict__ ws, int G, bf16* __restrict__ out, float* __restrict__ lse) {
  __shared__ int first[J4_MAX + 1];  // rows of the items before each CTA's
  __shared__ float4 osum[J4_WARPS][KVL / 4];
  __shared__ float tsum[J4_WARPS];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, l = tid & 31, warp = tid >> 5;
  const A4Rec* recs = reinterpret_cast<const A4Rec*>(ws);
  for (int i = tid; i < G; i += J4_THREADS) {
    const A4Rec r = recs[i];
    first[i + 1] = r.last < 0 ? 0 : r.nrows;
  }
  __syncthreads();
  if (warp == 0) {  // prefix sums
    int run = 0;
    for (int i = 0; i < G; i += 32) {
      int x = i + l < G ? first[i + l + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(FULL, x, o);
        if (l >= o) x += y;
      }
      if (i + l < G) first[i + l + 1] = run + x;
      run += __shfl_sync(FULL, x, 31);
    }
    if (l == 0) first[0] = 0;
  }
  __syncthreads();
  const int rows = first[G], ctas = gridDim.x;
  const int per = rows <= ctas ? 16 : rows <= 4 * ctas ? 4 : 1;  // warps a row
  const int grp = warp / per, in = warp % per, at_once = J4_WARPS / per;
  const u8* parts = ws + (size_t)G * sizeof(A4Rec);
  for (int w0 = blockIdx.x * at_once; w0 < rows; w0 += ctas * at_once) {
    const int w = w0 + grp;
    const bool live = w < rows;
    float4 o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    float t = 0.f, m = A4_LOW;
    long long row = 0;
    if (live) {
      int b = 0, e = G;  // the item: the last CTA with first[b] <= w
      while (e - b > 1) {
        const int mid = (b + e) / 2;
        if (first[mid] <= w) b = mid;
        else e = mid;
      }
      const A4Rec rec = recs[b];
      const int r = w - first[b], n = rec.last - b + 1;
      row = rec.row0 + r;
      auto part = [&](int i) {
        return reinterpret_cast<const float*>(parts + (size_t)(i == 0 ? 2 * b + 1 : 2 * (b + i)) * A4_PART);
      };
      for (int i = l; i < n; i += 32) {  // a part whose tokens the row does not see has no say
        const float* st = part(i) + A4_ROWS * KVL;
        if (st[A4_ROWS + r] != 0.f) m = fmaxf(m, st[r]);
      }
      m = warp_max(m);
#pragma unroll 2
      for (int i = in; i < n; i += per) {
        const float* p = part(i);
        const float pm = p[A4_ROWS * KVL + r], pt = p[A4_ROWS * (KVL + 1) + r];
        float4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = reinterpret_cast<const float4*>(p + r * KVL)[32 * j + l];
        const float wt = pt == 0.f ? 0.f : a4_exp2(pm - m);
        t = __fmaf_rn(wt, pt, t);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[j].x = __fmaf_rn(wt, v[j].x, o[j].x), o[j].y = __fmaf_rn(wt, v[j].y, o[j].y);
          o[j].z = __fmaf_rn(wt, v[j].z, o[j].z), o[j].w = __fmaf_rn(wt, v[j].w, o[j].w);
        }
      }
    }
    if (per > 1) {
      __syncthreads();  // the rows before have been read
#pragma unroll
      for (int j = 0; j < 4; ++j) osum[warp][32 * j + l] = o[j];
      if (l == 0) tsum[warp] = t;
      __syncthreads();
      if (in == 0) {
        for (int k = 1; k < per; ++k) {
          t += tsum[warp + k];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 v = osum[warp + k][32 * j + l];
            o[j].x += v.x, o[j].y += v.y, o[j].z += v.z, o[j].w += v.w;
          }
        }
      }
    }
    if (live && in == 0) {
      const float inv = t > 0.f ? 1.f / t : (t == 0.f ? 0.f : t);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint2 v;
        v.x = pack_bf16x2(o[j].x * inv, o[j].y * inv), v.y = pack_bf16x2(o[j].z * inv, o[j].w * inv);
        reinterpret_cast<uint2*>(out + row * KVL)[32 * j + l] = v;
      }
      if (l == 0) lse[row] = t == 0.f ? -INFINITY : (m + log2f(t)) * 0.6931471805599453f;
    }
  }
}

}  // namespace glmkv

// Attention of a packed call's rows over their sequences' 4-bit cache, causal among the fresh rows.
//   persistent: grid = SMs, block 384, dynamic smem A4_SMEM (222,208 B); glm_kv4_join follows
extern "C" __global__ void __launch_bounds__(glmkv::A4_THREADS, 1)
    glm_kv4_attn(const __grid_constant__ glmkv::A4Args a) {
  glmkv::a4_run<glmkv::A4_ATTN>(a);
}
// The same over each row's picked slots.
extern "C" __global__ void __launch_bounds__(glmkv::A4_THREADS, 1)
    glm_kv4_attn_picks(const __grid_constant__ glmkv::A4Args a) {
  glmkv::a4_run<glmkv::A4_PICKS>(a);
}
// Every cached token's weight added to acc. Same launch, no join.
extern "C" __global__ void __launch_bounds__(glmkv::A4_THREADS, 1)
    glm_kv4_weights(const __grid_constant__ glmkv::A4Args a) {
  glmkv::a4_run<glmkv::A4_WEIGHTS>(a);
}
// The split items of glm_kv4_attn and glm_kv4_attn_picks. grid: 2 x SMs (any), block 512
extern "C" __global__ void __launch_bounds__(glmkv::J4_THREADS)
    glm_kv4_join(const glmkv::u8* __restrict__ ws, int G, glmkv::bf16* __restrict__ out, float* __restrict__ lse) {
  glmkv::a4_join(ws, G, out, lse);
}
