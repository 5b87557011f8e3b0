// Attention of ragged chunks of new tokens over the paged KV cache: prompts in chunks, plain decode (one new token per
// request), and steps that mix the two.  Query i of a request with n keys and m new tokens sees keys 0 .. n - m + i.
//
//   o = sigmoid(gate) * sum_j w_j v_j / sum_j w_j,   w_j = 2^((q . k_j - m) scale log2 e)
//
// in one pass over the pages: the running maximum m moves only when a page exceeds it by more than AX_TAU (log2), the row
// sums and the accumulator are fp32, and the partial (o, m, l) of ranges that were cut are merged in page order.
//
// Rows.  The query heads of one kv head share its keys, so a tile's 128 rows are (token, head of the group) pairs of one
// request: 128 / group tokens at a time.  Q . K^T and P . V run on tcgen05 with the rows on the M side; a softmax thread
// owns a whole row of a page's scores, so its maximum and sum need no exchange, and the running maximum passes from the
// warp of one page to the warp of the next.
//
// P in 8 bits.  With e4m3 pages V is the B operand of an 8-bit MMA as it lies in the page, which saves the conversion
// of V to f16 (64 KB of shared memory and three passes over it per page) at the tensor time of one 16-bit product: P is
// given in two terms, an e5m2 value h of P 2^AX_BIAS and the e4m3 value of the remainder P 2^AX_BIAS - h.  h is within
// 2^(e-3) of a probability in [2^e, 2^(e+1)) and the remainder's own rounding within 2^(e-8): half a step of 2^-8, what
// bf16 has.  The range: the remainder is a normal number for probabilities down to 2^-11 of the maximum, h alone down to
// 2^-22 and, as a subnormal, 2^-25.  With bf16 pages P is bf16.  Error against 64 bits, 2-norm: 2.1e-3 (e4m3) and 2.3e-3
// (bf16), of which the output's own rounding to bf16 is 1.7e-3.
//
// Work.  Every (kv head, request, tile) costs its pages plus AX_OVH; the sequence of all of them is cut into equal
// ranges, one per CTA, so that a batch of any shape fills the GPU.  Every CTA finds its range from the lengths by itself
// (a closed form for the pages of a request's first k tiles), so nothing is planned on the host and a captured graph may
// be replayed with other lengths.
//
// What bounds it.  Prompts: a page costs the tensor pipe 1536 cycles (D = 256, e4m3: 512 for the scores, 1024 for the two
// terms of P . V) and takes about 2150.  The score buffers are the link: they and the accumulator fill the 512 columns of
// TMEM, so the scores of page t + NS wait for P . V of page t, and half of (softmax of a page, about 2600 cycles, + P . V,
// scores and hand-overs, about 1700) is what a page takes with two buffers.  The exponential unit is busy 1024 of those.
// Four 2048-token chunks behind 6144 tokens: 0.60 ms at first and 0.70 ms sustained (1545 MHz under the power limit),
// 1.4 PFLOP/s.  Decode: 64 requests x 8192 tokens, 0.54 GB of e4m3 pages: 100 us, 107 us sustained (1440 MHz) = 5.0 TB/s.
// Tried and dropped: four softmax warps per scheduler, each with half of a page (607 -> 650 us: more instructions, no
// shorter chain); a quarter of the exponentials as a cubic on the FMA pipe (605 -> 610 us); polling instead of suspended
// waits (650 -> 687 us: the pollers take the issue slots); 8 x 8 exchanges between lanes for an epilogue that writes whole
// lines (mixed step 106 -> 119 us).
#include "common.cuh"
#include "host.h"

namespace b200 {

B200_DEFINE_WAIT_BUDGET_SETTER(set_wait_budget_attn_extend)

constexpr int AX_PAGE = 128;
constexpr int AX_OVH = 4;              // cost of a tile beside its pages, in pages (a mixed step with 2 / 4 / 6 / 8: 118 / 96 /
                                       // 94 / 100 us; chunks of 1000 to 1500 bf16 tokens: 104 / 106 / 108 / 128 us)
constexpr int AX_MIN_UNITS = 2;        // smallest range worth a CTA of its own (one token, 8192 keys, with 1 / 2 / 4: 25.8 / 19.7 /
                                       // 20.3 us: more pieces cost the merge more than they save)
constexpr float AX_BIAS = 8.f;         // log2 scale of the 8-bit probabilities
constexpr float AX_TAU = 4.f;          // log2 distance that moves the running maximum: 2^(8 + 4) fits both formats
constexpr int AX_ITEMS = 4;            // ring of work items
constexpr int AX_WARPS = 12;           // K, V, MMA, scheduler, 8 softmax
constexpr int AX_THREADS = AX_WARPS * 32;
constexpr int AX_SOFT0 = 4, AX_SOFT = 8;

struct AxArgs {
  const bf16* gate;
  long long gate_stride;
  const void* vc;
  int num_pages;
  const int32_t* table;
  int pt_stride;
  const int32_t* cu;
  const int32_t* seqlens;
  int B, T, hq, hkv, grp, tpt;   // grp query heads per kv head, tpt tokens per tile
  float scale_log2;
  bf16* out;
  int32_t* desc;                 // [grid][8]: tiles to merge
  float* part;                   // [2 * grid][D / 4][rows][4] unnormalised, then [2 * grid][2][rows]: maximum, row sum
  int rows;                      // tpt * grp
  int sub;                       // tokens of a small Q box: their rows fill whole groups of 8
  int32_t* status;
};

// one piece of work: pages [p0, p1) of one tile
struct AxItem {
  int req, head, tok0, ntok;     // tok0: row of the tile's first token in q
  int pos0, p0, p1, slot;        // pos0: its place in the request; slot: partial slot or -1
};

// the first of an item's pages that not every row of its tile sees to the end
__device__ __forceinline__ int ax_first_edge(const AxItem& x) { return max(x.p0, (max(x.pos0, -1) + 1) / AX_PAGE); }

template <bool F8, int D>
struct AxShape {
  static constexpr int ES = F8 ? 1 : 2;
  static constexpr int ROWB = D * ES;                  // bytes of a Q or K row
  static constexpr int NB = ROWB / 128;                // 128-byte blocks of a row
  static constexpr int PAGEB = AX_PAGE * ROWB;         // bytes of a K (or V) page of one kv head
  static constexpr int UNIT = PAGEB < 32768 ? PAGEB : 32768;
  static constexpr int PU = PAGEB / UNIT;              // ring units per page
  static constexpr int NK = PU == 2 ? 2 : (UNIT == 16384 ? 5 : 3);   // K stages (units)
  static constexpr int NV = PU == 2 ? 3 : (UNIT == 16384 ? 5 : 3);   // V stages
  static constexpr int QB = NB * 16384;                // Q tile: NB blocks of [128 rows x 128 bytes]
  static constexpr int OFF_K = QB;
  static constexpr int OFF_V = OFF_K + NK * UNIT;
  static constexpr int OFF_BAR = OFF_V + NV * UNIT;
  static constexpr int OFF_ITEM = OFF_BAR + 640;       // barriers and 40 bytes
  static constexpr int OFF_RED = OFF_ITEM + AX_ITEMS * 32;
  static constexpr int SMEM = OFF_RED + 2 * 2 * 128 * 4;
  static_assert(SMEM <= 232448, "shared memory of a CTA");
  static constexpr int VBOX = D * 128;                 // one V box: D rows of 128 bytes
  static constexpr int NS = D == 128 ? 3 : 2;          // score buffers: what the accumulator leaves of 512 columns
  static_assert((2 * NK + 3 * NV + 3 * AX_ITEMS + 6 * NS + 14) * 8 + 40 <= 640, "room for the barriers");
};

__device__ __forceinline__ uint32_t ax_sw128(int row, int chunk) {
  return static_cast<uint32_t>((row >> 3) * 1024 + (row & 7) * 128 + ((chunk ^ (row & 7)) << 4));
}
// Shared-memory descriptors of 128-byte-swizzled K-major tiles differ in their low word only (umma_desc_sw128).  The MMAs are
// issued by one elected lane of a warp whose control flow is uniform, from low words that are a base plus a constant: the
// operands then stay in uniform registers.  Issued by a lane of a divergent branch with 64-bit descriptors built in place, an
// MMA took 150 cycles of issue whatever its size; so it takes 64 (N = 128) and 128 (N = 256), the tensor pipe's own time.
constexpr uint32_t AX_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t ax_desc_lo(uint32_t smem_addr) { return ((smem_addr & 0x3ffffu) >> 4) | (1u << 16); }
// D += A B, A in tensor memory
template <bool F8>
__device__ __forceinline__ void ax_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  if (F8)
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 b, {%2, %5};\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], b, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(AX_DESC_HI)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 b, {%2, %5};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(AX_DESC_HI)
        : "memory");
}
// D += A B, both in shared memory
template <bool F8>
__device__ __forceinline__ void ax_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  if (F8)
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 a, {%1, %5};\nmov.b64 b, {%2, %5};\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n}\n" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(AX_DESC_HI)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 a, {%1, %5};\nmov.b64 b, {%2, %5};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(AX_DESC_HI)
        : "memory");
}
// instruction descriptor: M = 128, N = n, fp32 accumulator, K-major operands
__host__ __device__ constexpr uint32_t ax_idesc(uint32_t a_fmt, uint32_t b_fmt, uint32_t n) {
  return (UMMA_C_F32 << 4) | (a_fmt << 7) | (b_fmt << 10) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void ax_tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void ax_tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ax_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two probabilities (f16 pair) to their e5m2 values, in the upper byte of each half: rounded to three significant bits (ties
// away), which leaves an f16 whose lower byte is zero
__device__ __forceinline__ uint32_t ax_head(uint32_t h) { return (h + 0x00800080u) & 0xff00ff00u; }
__device__ __forceinline__ uint32_t ax_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// e4m3 of the (exact) difference of two f16 pairs, in the low half
__device__ __forceinline__ uint32_t ax_rest(uint32_t h, uint32_t head) {
  uint32_t d;
  uint16_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(h), "r"(head));
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(d));
  return r;
}
__device__ __forceinline__ float ax_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// (a, b) <- (a, b) * m + c and (a, b) <- (a, b) + (c, d), two fp32 lanes per instruction
__device__ __forceinline__ void ax_fma2(float& a, float& b, float m, float c) {
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %2};\nmov.b64 z, {%3, %3};\n"
      "fma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}\n"
      : "+f"(a), "+f"(b)
      : "f"(m), "f"(c));
}
__device__ __forceinline__ void ax_add2(float& a, float& b, float c, float d) {
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %3};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}
__device__ __forceinline__ void ax_tma_load_3d(void* smem_dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(smem_u32(smem_dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// sum over i < m of floor((a + i s) / d); s <= 128, d <= 128, m <= 2^24 (Euclid's descent on (d, s); every divide in 32 bits)
__device__ __forceinline__ long long ax_floor_sum(uint32_t m, uint32_t d, uint32_t s, uint32_t a) {
  long long r = 0;
  while (m > 0) {
    r += static_cast<long long>(m) * (a / d);
    a %= d;
    r += static_cast<long long>(m) * (m - 1) / 2 * (s / d);
    s %= d;
    const uint32_t y = s * m + a;
    if (y < d) break;
    m = y / d;
    a = y % d;
    const uint32_t t = d;
    d = s;
    s = t;
  }
  return r;
}
// x / y, in 32 bits where both fit.  This and the costs below stay out of line: a CTA runs them a few times at its start, when
// every instruction line is a miss
__device__ __noinline__ long long ax_div(long long x, long long y) {
  if (((x | y) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
  return x / y;
}
// pages that a tile reads whose last token sees keys 0 .. end - 1
__device__ __forceinline__ int ax_pages(int end) { return end <= 0 ? 0 : (end + AX_PAGE - 1) / AX_PAGE; }
// cost of a request's first k tiles, all of tpt tokens; ctx: keys before its first new token (negative: missing)
__device__ __noinline__ long long ax_cost(int k, int ctx, int tpt) {
  const int skip = ctx < 0 ? min(k, -ctx / tpt) : 0;   // tiles whose last token sees nothing
  return static_cast<long long>(k) * AX_OVH +
         ax_floor_sum(k - skip, AX_PAGE, tpt, static_cast<uint32_t>(ctx + (skip + 1) * tpt + AX_PAGE - 1));
}
__device__ __forceinline__ long long ax_cost_all(int n, int ctx, int tpt) {
  if (n <= 0) return 0;
  return ax_cost((n - 1) / tpt, ctx, tpt) + AX_OVH + ax_pages(ctx + n);
}

// mask of the first n bytes of a word
__device__ __forceinline__ uint32_t ax_below(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : ~0u >> (32 - n * 8); }
// mask of the e4m3 or bf16 elements of a word that are NaN or infinite
template <bool F8>
__device__ __forceinline__ uint32_t ax_not_finite(uint32_t w) {
  return F8 ? ((((w & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u) * 0xffu
            : ((((w & 0x7f807f80u) + 0x00800080u) >> 15) & 0x00010001u) * 0xffffu;
}

// Request b: its rows lo .. lo + n - 1 and the keys before its first new token, from lengths that may be anything: rows are kept
// inside [0, T), keys behind the block table are missing anyway and do not count
__device__ __forceinline__ void ax_request(const AxArgs& p, int b, int& lo, int& n, int& ctx) {
  lo = min(max(p.cu[b], 0), p.T);
  n = min(max(p.cu[b + 1], 0), p.T) - lo;
  ctx = min(max(p.seqlens[b], 0) - n, p.pt_stride * AX_PAGE);
}

// What is not finite in the V of the keys that were cleared for a tile goes back to a row that sees them: NaN, or an infinity
// of either sign, in the columns where it stood.  Runs for the tiles that hold such a value only.
template <bool F8, int D>
__device__ __forceinline__ void ax_give_back(const AxArgs& p, const AxItem& x, int row, int lim, long long tok, int hd, int col0) {
  asm volatile("" ::: "memory");
#pragma unroll 1
  for (int d = col0; d < col0 + D / 2; ++d) {
    float odd = 0.f;
#pragma unroll 1
    for (int j = max(x.pos0 + 1, x.p0 * AX_PAGE); j <= min(lim, x.p1 * AX_PAGE - 1); ++j) {
      const int id = j / AX_PAGE < p.pt_stride ? p.table[static_cast<size_t>(x.req) * p.pt_stride + j / AX_PAGE] : -1;
      if (id < 0 || id >= p.num_pages) continue;
      const size_t at = ((static_cast<size_t>(id) * p.hkv + x.head) * D + d) * AX_PAGE + j % AX_PAGE;
      if (F8) {
        if ((static_cast<const uint8_t*>(p.vc)[at] & 0x7f) == 0x7f) odd = __int_as_float(0x7fffffff);
      } else {
        const float v = bf2f(static_cast<const bf16*>(p.vc)[at]);
        if (!isfinite(v)) odd += v;
      }
    }
    if (odd == 0.f) continue;
    // added to what this thread has just stored there, which may be infinite already
    if (x.slot >= 0) {
      float* o = p.part + ((static_cast<size_t>(x.slot) * (D / 4) + d / 4) * p.rows + row) * 4 + d % 4;
      *o = __ldcg(o) + odd;
    } else {
      if (p.gate) odd = odd / (1.f + __expf(-bf2f(p.gate[tok * p.gate_stride + static_cast<long long>(hd) * D + d])));
      unsigned short* o = reinterpret_cast<unsigned short*>(p.out + (tok * p.hq + hd) * D + d);
      *o = __bfloat16_as_ushort(f2bf(bf2f(__ushort_as_bfloat16(__ldcg(o))) + odd));
    }
  }
}

// Waits of a whole warp: every lane polls, and all give up together.  The wait proper stays out of line: most barriers are
// complete when they are asked for, and the MMA issuer's own instructions have to fit between its MMAs.
__device__ __noinline__ bool ax_wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  return __all_sync(FULL_MASK, mbar_wait(bar, parity, abort_flag, status, code));
}
__device__ __forceinline__ bool ax_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (__all_sync(FULL_MASK, mbar_try(bar, parity))) return true;
  return ax_wait_slow(bar, parity, abort_flag, status, code);
}
__device__ __forceinline__ bool ax_test(uint64_t* bar, uint32_t parity) {   // without waiting
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// After an abandoned wait: gives a copy or a commit that is still in flight a bounded time.
__device__ __forceinline__ void ax_drain(uint64_t* bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer();
  while (!mbar_try(bar, parity) && globaltimer() - t0 < 20ull * 1000 * 1000) {
  }
}

template <bool F8, int D>
__global__ void __launch_bounds__(AX_THREADS, 1)
attn_extend_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQs,
                   const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const AxArgs p) {
  using X = AxShape<F8, D>;
  extern __shared__ __align__(1024) uint8_t smem[];   // the swizzled tiles start on 1024 bytes; there is no room for slack
  if (smem_u32(smem) & 1023u) {
    pdl_wait();
    if (threadIdx.x == 0) {
      p.desc[blockIdx.x * 8] = 0;
      if (p.status) atomicCAS(p.status, 0, ST_WAIT_STATE);
    }
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + X::OFF_BAR);
  uint64_t* kfull = bars;                 // [NK]
  uint64_t* kempty = kfull + X::NK;       // [NK]
  uint64_t* vfull = kempty + X::NK;       // [NV]
  uint64_t* vempty = vfull + X::NV;       // [NV]
  uint64_t* ifull = vempty + X::NV;       // [AX_ITEMS] item written
  uint64_t* iempty = ifull + AX_ITEMS;    // [AX_ITEMS] all roles are done with it
  uint64_t* sfull = iempty + AX_ITEMS;    // [NS] scores complete in TMEM
  uint64_t* pready = sfull + X::NS;       // [NS][4 quarters] probabilities written (and O rescaled if needed)
  uint64_t* mpub = pready + 4 * X::NS;    // [2 page parities][4 quadrants] running maximum published
  uint64_t* lpub = mpub + 8;              // [4] both warps' row sums published, the last P . V done
  uint64_t* qfull = lpub + 4;             // Q tile landed
  uint64_t* qempty = qfull + 1;           // the item's last score MMA is done
  uint64_t* pvdone = qempty + 1;          // [NS] P . V of a page done
  uint64_t* ofree = pvdone + X::NS;       // [AX_ITEMS] the item's accumulator has been read (by ring place: a warp without rows
                                          // may be some items ahead, and must not arrive twice in one phase)
  uint64_t* vtail = ofree + AX_ITEMS;     // [NV] V page that has to be tended landed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(vtail + X::NV);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_start = reinterpret_cast<int*>(tmem_slot + 2);   // request
  long long* s_off = reinterpret_cast<long long*>(tmem_slot + 4);
  volatile int* s_odd = reinterpret_cast<volatile int*>(tmem_slot + 6);   // [AX_ITEMS] values that are not finite were cleared
  AxItem* items = reinterpret_cast<AxItem*>(smem + X::OFF_ITEM);
  float* s_m = reinterpret_cast<float*>(smem + X::OFF_RED);   // [2 page parities][128 rows] running maximum
  float* s_l = s_m + 256;                                     // [2 page parities][128 rows] row sum
  long long* s_scan = reinterpret_cast<long long*>(smem + X::OFF_V);   // prelude only, before any copy is issued

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < X::NK; ++i) {
      mbar_init(&kfull[i], 1);
      mbar_init(&kempty[i], 1);
    }
    for (int i = 0; i < X::NV; ++i) {
      mbar_init(&vfull[i], 1);
      mbar_init(&vempty[i], 1);
      mbar_init(&vtail[i], 1);
    }
    for (int i = 0; i < AX_ITEMS; ++i) {
      mbar_init(&ifull[i], 1);
      mbar_init(&iempty[i], 3 + AX_SOFT);   // K, V, MMA, softmax warps
      mbar_init(&ofree[i], AX_SOFT);
    }
    for (int i = 0; i < X::NS; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pvdone[i], 1);
    }
    for (int i = 0; i < 4 * X::NS; ++i) mbar_init(&pready[i], AX_SOFT / 2);
    for (int i = 0; i < 4; ++i) mbar_init(&lpub[i], 2);
    for (int i = 0; i < 8; ++i) mbar_init(&mpub[i], 1);
    mbar_init(qfull, 1);
    mbar_init(qempty, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 2) tmem_alloc(tmem_slot, 512);
  for (int i = threadIdx.x; i < X::QB / 16; i += AX_THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  pdl_wait();
  pdl_launch();

  // ---- this CTA's range of the work: every thread costs a slice of the requests, the CTA scans the slices ----
  const int cta = blockIdx.x, grid = gridDim.x;
  const int per = (p.B + AX_THREADS - 1) / AX_THREADS, b0 = min(p.B, static_cast<int>(threadIdx.x) * per), b1 = min(p.B, b0 + per);
  long long mine = 0;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    int lo, n, ctx;
    ax_request(p, b, lo, n, ctx);
    mine += ax_cost_all(n, ctx, p.tpt);
  }
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(FULL_MASK, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) s_scan[warp] = inc;
  if (threadIdx.x == 0) *s_start = -1;
  __syncthreads();
  long long before = inc - mine, C = 0;
  for (int w = 0; w < AX_WARPS; ++w) {
    const long long v = s_scan[w];
    if (w < warp) before += v;
    C += v;
  }
  const long long U = C * p.hkv;
  // n_eff ranges: the first `more` of them have `each` + 1 units, the others `each`
  const int n_eff = U >= static_cast<long long>(grid) * AX_MIN_UNITS ? grid : static_cast<int>((U + AX_MIN_UNITS - 1) / AX_MIN_UNITS);
  const long long each = n_eff ? ax_div(U, n_eff) : 0;
  const int more = static_cast<int>(U - each * n_eff);
  auto bound = [&](int c) -> long long { return c * each + min(c, more); };
  auto range_of = [&](long long u) -> int {   // the range that holds unit u
    const long long lo = more * (each + 1);
    return static_cast<int>(u < lo ? ax_div(u, each + 1) : more + ax_div(u - lo, each));
  };
  const long long u0 = cta < n_eff ? bound(cta) : U, u1 = cta < n_eff ? bound(cta + 1) : U;
  const int head0 = u0 < u1 ? static_cast<int>(ax_div(u0, C)) : 0;
  if (u0 < u1) {
    const long long v0 = u0 - head0 * C;
    if (v0 >= before && v0 < before + mine) {
      long long at = before;
      int b = b0;
#pragma unroll 1
      for (; b < b1 - 1; ++b) {      // the last one needs no look
        int lo, n, ctx;
        ax_request(p, b, lo, n, ctx);
        const long long c = ax_cost_all(n, ctx, p.tpt);
        if (v0 < at + c) break;
        at += c;
      }
      *s_start = b;
      *s_off = v0 - at;
    }
  }
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(FULL_MASK, *tmem_slot, 0);
  const uint32_t TM_O = tmem, TM_S = tmem + 512 - X::NS * 128;   // O: D columns; NS score buffers of 128

  // items in order; `it` counts them
  auto item_wait = [&](int it, AxItem& x) -> bool {
    if (!ax_wait(&ifull[it % AX_ITEMS], (it / AX_ITEMS) & 1, abort_flag, p.status, ST_WAIT_FULL)) return false;
    x = items[it % AX_ITEMS];
    return x.p1 > x.p0;    // an empty item ends the list
  };
  auto item_done = [&](int it) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&iempty[it % AX_ITEMS]);
  };

  if (warp == 3) {
    // ---------------- scheduler: walks the tiles of this CTA's range.  The same warp tends the copies of the V pages that not
    // every row of their tile sees to the end.  A zero probability times a NaN or an infinity would spoil a row, so the places
    // behind the last key are cleared (they may hold anything), and so is what is not finite in the keys that some rows see
    // and others do not; the epilogue then gives it back to the rows that see it.  Such a page lands on a barrier of its own
    // and counts as full once it is tended; it is tended whenever it lands, also while a place in the item ring is waited for
    int it = 0, cl = 0, ce = 0, cu = 0, pages = 0;   // items written; items tended, pages and units of the next; their pages
    uint32_t tails = 0;                      // per stage: phase of its tail barrier
    bool ok = true, described = false;
    auto tend = [&]() -> bool {              // the next such unit, if it has landed
      if (cl == it) return false;
      const AxItem x = items[cl % AX_ITEMS];
      const int j = ax_first_edge(x) + ce;
      if (j < x.p1) {
        const int st = ((pages + j - x.p0) * X::PU + cu) % X::NV;
        if (!__all_sync(FULL_MASK, ax_test(&vtail[st], (tails >> st) & 1))) return false;
        tails ^= 1u << st;
        uint32_t found = 0;
#pragma unroll 1
        for (int c = 0; c < X::UNIT / X::VBOX; ++c) {
          // bytes of a row of the box: from `lo` on not every row of the tile sees them, from `hi` on none does
          const int at = j * AX_PAGE * X::ES + (cu * (X::UNIT / X::VBOX) + c) * 128;
          const int lo = min(128, max(0, (x.pos0 + 1) * X::ES - at)), hi = min(128, max(0, (x.pos0 + x.ntok) * X::ES - at));
          uint8_t* box = smem + X::OFF_V + st * X::UNIT + c * X::VBOX;
#pragma unroll 1
          for (int ch = lo >> 4; ch < 8; ++ch) {
            if (ch * 16 >= hi) {
#pragma unroll
              for (int d = 0; d < D; d += 32) *reinterpret_cast<uint4*>(box + ax_sw128(d + lane, ch)) = make_uint4(0, 0, 0, 0);
              continue;
            }
            uint32_t keep[4], look[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              keep[k] = ax_below(hi - ch * 16 - k * 4);
              look[k] = keep[k] & ~ax_below(lo - ch * 16 - k * 4);
            }
#pragma unroll 2
            for (int d = lane; d < D; d += 32) {
              uint4* w = reinterpret_cast<uint4*>(box + ax_sw128(d, ch));
              uint4 v = *w;
              uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t odd = ax_not_finite<F8>(e[k]) & look[k];
                found |= odd;
                e[k] &= keep[k] & ~odd;
              }
              *w = make_uint4(e[0], e[1], e[2], e[3]);
            }
          }
        }
        if (__any_sync(FULL_MASK, found != 0) && lane == 0) s_odd[cl % AX_ITEMS] = 1;
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&vfull[st]);
        if (++cu == X::PU) {
          cu = 0;
          ++ce;
        }
        return true;
      }
      ce = 0;
      pages += x.p1 - x.p0;
      ++cl;
      return true;
    };
    // tends the tails until `done` holds
    auto until = [&](auto done) -> bool {
      const unsigned long long t0 = globaltimer();
      while (true) {
        if (tend()) continue;
        if (done()) return true;
        __nanosleep(32);
        const bool late = globaltimer() - t0 > g_wait_budget_ns;
        if (__any_sync(FULL_MASK, *abort_flag || late)) {
          if (late) {
            *abort_flag = 1;
            if (p.status) atomicCAS(p.status, 0, ST_WAIT_EMPTY);
          }
          return false;
        }
      }
    };
    auto push = [&](const AxItem& x) -> bool {
      const int s = it % AX_ITEMS;
      const uint32_t ph = ((it / AX_ITEMS) & 1) ^ 1u;
      if (!until([&] { return cl + AX_ITEMS > it && __all_sync(FULL_MASK, ax_test(&iempty[s], ph)); })) return false;
      if (lane == 0) {
        items[s] = x;
        s_odd[s] = 0;
        mbar_arrive(&ifull[s]);
      }
      __syncwarp();
      ++it;
      return true;
    };
    if (u0 < u1) {
      const long long before_me = cta > 0 ? bound(cta - 1) : 0;
      int head = head0, b = *s_start, base = -32;
      long long off = *s_off, u = u0 - off;      // u: where the request's tiles begin
      int w_lo = 0, w_n = 0, w_ctx = 0;          // a window of 32 requests, one per lane
      while (ok && u < u1) {
        if (b >= p.B) {
          b = 0;
          ++head;
        }
        if (b < base || b >= base + 32 || base < 0) {
          base = b;
          ax_request(p, min(b + lane, p.B - 1), w_lo, w_n, w_ctx);
          if (b + lane >= p.B) w_n = 0;
        }
        const int lo = __shfl_sync(FULL_MASK, w_lo, b - base), n = __shfl_sync(FULL_MASK, w_n, b - base);
        const int ctx = __shfl_sync(FULL_MASK, w_ctx, b - base);
        if (n <= 0) {
          ++b;
          continue;
        }
        const int tiles = (n + p.tpt - 1) / p.tpt;
        int k = 0;
        if (off > 0) {                           // the first tile whose range reaches past `off`: 32 candidates a round
          int span = tiles;
          while (span > 1) {
            const int step = (span + 31) / 32;
            const bool under = lane * step < span && ax_cost(k + lane * step, ctx, p.tpt) <= off;
            const int l = 31 - __clz(__ballot_sync(FULL_MASK, under));
            k += l * step;
            span = min(step, span - l * step);
          }
        }
        long long ts = u + (off > 0 ? ax_cost(k, ctx, p.tpt) : 0);
        off = 0;
        for (; ok && k < tiles && ts < u1; ++k) {
          const int nt = min(p.tpt, n - k * p.tpt), end = ctx + k * p.tpt + nt, pg = ax_pages(end);
          const long long fp = ts + AX_OVH, te = fp + pg;
          if (pg == 0) {
            if (ts >= u0)                        // nobody sees anything: zero rows, written by the range that has the start
              for (int r = 0; r < nt; ++r) {
                uint4* o = reinterpret_cast<uint4*>(p.out + (static_cast<long long>(lo + k * p.tpt + r) * p.hq + head * p.grp) * D);
                if (lo + k * p.tpt + r < p.T)
                  for (int c = lane; c < p.grp * D / 8; c += 32) o[c] = make_uint4(0, 0, 0, 0);
              }
          } else {
            const long long a = max(fp, u0), z = min(te, u1);
            if (a < z) {
              AxItem x;
              x.req = b;
              x.head = head;
              x.tok0 = lo + k * p.tpt;
              x.ntok = nt;
              x.pos0 = ctx + k * p.tpt;
              x.p0 = static_cast<int>(a - fp);
              x.p1 = static_cast<int>(z - fp);
              x.slot = x.p0 == 0 ? (x.p1 == pg ? -1 : 2 * cta + 1) : 2 * cta;
              if (x.p0 > 0 && fp >= before_me) {     // the first cut of its tile: merged in this CTA's name
                described = true;
                if (lane == 0) {
                  int32_t* d = p.desc + cta * 8;
                  d[0] = te <= u1 ? 2 : range_of(te - 1) - cta + 2;   // pieces
                  d[1] = x.tok0;
                  d[2] = nt;
                  d[3] = head;
                }
              }
              ok = push(x);
            }
          }
          ts = te;
        }
        u = ts;
        ++b;
      }
    }
    if (!described && lane == 0) p.desc[cta * 8] = 0;
    if (ok) {
      AxItem end{};
      if (push(end)) until([&] { return cl == it; });
    }
  } else if (warp == 0) {
    // ---------------- K pages and Q tiles ----------------
    AxItem x;
    int un = 0, issued = 0;        // K units
    bool ok = true;
    int it = 0;
    for (; ok && item_wait(it, x); ++it) {
      if (it > 0) ok = ax_wait(qempty, (it - 1) & 1, abort_flag, p.status, ST_WAIT_EMPTY);
      if (!ok) break;
      if (lane == 0) {
        // A tile of few tokens gets only their rows: the others stay zero (or an earlier item's), and products of zeros take less
        // power, which is what limits the clock here (64 x 8192 tokens of decode, sustained: 117 us with full boxes, 114 so)
        const int boxes = (x.ntok + p.sub - 1) / p.sub;
        if (boxes * p.sub * 2 <= p.tpt) {
          mbar_expect_tx(qfull, X::NB * boxes * p.sub * p.grp * 128);
          for (int t = 0; t < boxes; ++t)
            for (int c = 0; c < X::NB; ++c)
              ax_tma_load_3d(smem + c * 16384 + t * p.sub * p.grp * 128, &tmQs, c * 128, x.head * p.grp, x.tok0 + t * p.sub, qfull);
        } else {
          mbar_expect_tx(qfull, X::NB * p.rows * 128);
          for (int c = 0; c < X::NB; ++c) ax_tma_load_3d(smem + c * 16384, &tmQ, c * 128, x.head * p.grp, x.tok0, qfull);
        }
      }
      int ids = 0;
      for (int j = x.p0; ok && j < x.p1; ++j) {
        if (((j - x.p0) & 31) == 0) {
          const int e = j + lane;
          ids = e < x.p1 && e < p.pt_stride ? p.table[static_cast<size_t>(x.req) * p.pt_stride + e] : -1;
          if (e < x.p1 && (ids < 0 || ids >= p.num_pages)) {
            if (p.status) atomicCAS(p.status, 0, B200_ST_BAD_PAGE);
            ids = p.num_pages;     // behind the pool: the copy fills zeros
          }
        }
        const int id = __shfl_sync(FULL_MASK, ids, (j - x.p0) & 31);
        const int y = id >= p.num_pages ? p.num_pages * p.hkv * AX_PAGE : (id * p.hkv + x.head) * AX_PAGE;
        for (int u = 0; u < X::PU; ++u, ++un) {
          const int st = un % X::NK;
          ok = ax_wait(&kempty[st], ((un / X::NK) & 1) ^ 1u, abort_flag, p.status, ST_WAIT_EMPTY);
          if (!ok) break;
          if (lane == 0) {
            mbar_expect_tx(&kfull[st], X::UNIT);
            for (int c = 0; c < X::UNIT / 16384; ++c)
              tma_load_2d(smem + X::OFF_K + st * X::UNIT + c * 16384, &tmK, (u * (X::UNIT / 16384) + c) * 128, y, &kfull[st]);
          }
          issued = un + 1;
        }
      }
      if (ok) item_done(it);
    }
    if (*abort_flag && lane == 0) {
      for (int i = max(0, issued - X::NK); i < issued; ++i) ax_drain(&kfull[i % X::NK], (i / X::NK) & 1);
      ax_drain(qfull, it & 1);
    }
  } else if (warp == 1) {
    // ---------------- V pages ----------------
    AxItem x;
    int un = 0, issued = 0;
    bool ok = true;
    for (int it = 0; ok && item_wait(it, x); ++it) {
      int ids = 0;
      for (int j = x.p0; ok && j < x.p1; ++j) {
        if (((j - x.p0) & 31) == 0) {
          const int e = j + lane;
          ids = e < x.p1 && e < p.pt_stride ? p.table[static_cast<size_t>(x.req) * p.pt_stride + e] : -1;
        }
        const int id = __shfl_sync(FULL_MASK, ids, (j - x.p0) & 31);
        const int y = id < 0 || id >= p.num_pages ? p.num_pages * p.hkv * D : (id * p.hkv + x.head) * D;
        uint64_t* full = j >= ax_first_edge(x) ? vtail : vfull;
        for (int u = 0; u < X::PU; ++u, ++un) {
          const int st = un % X::NV;
          ok = ax_wait(&vempty[st], ((un / X::NV) & 1) ^ 1u, abort_flag, p.status, ST_WAIT_EMPTY);
          if (!ok) break;
          if (lane == 0) {
            mbar_expect_tx(&full[st], X::UNIT);
            for (int c = 0; c < X::UNIT / X::VBOX; ++c)
              tma_load_2d(smem + X::OFF_V + st * X::UNIT + c * X::VBOX, &tmV, (u * (X::UNIT / X::VBOX) + c) * 128, y, &full[st]);
          }
          issued = un + 1;
        }
      }
      if (ok) item_done(it);
    }
    if (*abort_flag && lane == 0)   // a page on its tail barrier never counts as full now: its time runs out instead
      for (int i = max(0, issued - X::NV); i < issued; ++i) ax_drain(&vfull[i % X::NV], (i / X::NV) & 1);
  } else if (warp == 2) {
    // ---------------- MMA issuer.  The score MMAs run NS pages ahead of the P . V MMAs (also into the next item), so the
    // tensor pipe has a product to do while the softmax warps work on a page.  P . V is issued per quarter of a page, as
    // its probabilities arrive ----------------
    const uint32_t q_lo = ax_desc_lo(smem_u32(smem)), k_lo = ax_desc_lo(smem_u32(smem + X::OFF_K)),
                   v_lo = ax_desc_lo(smem_u32(smem + X::OFF_V));
    constexpr uint32_t id_s = ax_idesc(F8 ? 0u : 1u, F8 ? 0u : 1u, 128);
    constexpr uint32_t id_hi = ax_idesc(1u, F8 ? 0u : 1u, D);     // P: e5m2 or bf16 (both 1); V: e4m3 0 or bf16 1
    constexpr uint32_t id_lo = ax_idesc(0u, 0u, D);
    auto get = [&](int it, int& n) -> bool {       // pages of item `it`
      if (!ax_wait(&ifull[it % AX_ITEMS], (it / AX_ITEMS) & 1, abort_flag, p.status, ST_WAIT_FULL)) return false;
      n = __shfl_sync(FULL_MASK, items[it % AX_ITEMS].p1 - items[it % AX_ITEMS].p0, 0);
      return n > 0;
    };
    int s_it = 0, s_i = 0, s_n = 0, s_b = 0, k_st = 0, k_ph = 0;
    bool s_more = true, ok = true;
    auto issue_s = [&]() {
      if (!s_more) return;
      if (s_i == s_n) {
        if (!get(s_it, s_n)) {
          s_more = false;
          return;
        }
        s_i = 0;
        if (!ax_wait(qfull, s_it & 1, abort_flag, p.status, ST_WAIT_FULL)) {
          s_more = ok = false;
          return;
        }
        ++s_it;
      }
      const uint32_t d = TM_S + s_b * 128;
#pragma unroll
      for (int u = 0; u < X::PU; ++u) {
        if (!ax_wait(&kfull[k_st], k_ph, abort_flag, p.status, ST_WAIT_FULL)) {
          s_more = ok = false;
          return;
        }
        tc_fence_after();
        const uint32_t kb = k_lo + k_st * (X::UNIT >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < X::UNIT / 16384 * 4; ++kk) {     // 32 bytes of a row per step, four steps per 128-byte block
            const int c = kk >> 2;
            ax_mma_ss<F8>(d, q_lo + (u * (X::UNIT / 16384) + c) * 1024 + (kk & 3) * 2, kb + c * 1024 + (kk & 3) * 2, id_s,
                          (u | kk) != 0);
          }
          tc_commit(&kempty[k_st]);
          if (u == X::PU - 1) {
            tc_commit(&sfull[s_b]);
            if (s_i == s_n - 1) tc_commit(qempty);
          }
        }
        __syncwarp();
        if (++k_st == X::NK) {
          k_st = 0;
          k_ph ^= 1;
        }
      }
      s_b = s_b + 1 == X::NS ? 0 : s_b + 1;
      ++s_i;
    };
#pragma unroll 1
    for (int i = 0; i < X::NS; ++i) issue_s();
    int it = 0, n = 0, b = 0, b_ph = 0, v_st = 0, v_ph = 0;
    while (ok && get(it, n)) {
      for (int i = 0; ok && i < n; ++i) {
        const uint32_t pa = TM_S + b * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c) {          // 32 keys each
          if (c == 0 || (X::PU == 2 && c == 2)) {
            ok = ax_wait(&vfull[v_st], v_ph, abort_flag, p.status, ST_WAIT_FULL);
            if (!ok) break;
          }
          ok = ax_wait(&pready[b * 4 + c], b_ph, abort_flag, p.status, ST_WAIT_TMEM_FULL);
          if (ok && c == 0 && i == 0 && it > 0)
            ok = ax_wait(&ofree[(it - 1) % AX_ITEMS], ((it - 1) / AX_ITEMS) & 1, abort_flag, p.status, ST_WAIT_TMEM_EMPTY);
          if (!ok) break;
          tc_fence_after();
          const uint32_t vb = v_lo + v_st * (X::UNIT >> 4);
          const bool unit_end = c == 3 || (X::PU == 2 && c == 1);
          if (elect_one()) {
            if (F8) {     // the values, then the remainders
              ax_mma_ts<F8>(TM_O, pa + c * 32, vb + c * 2, id_hi, (i | c) != 0);
              ax_mma_ts<F8>(TM_O, pa + c * 32 + 8, vb + c * 2, id_lo, 1);
            } else {      // 16 keys a step; a box holds 64 keys
#pragma unroll
              for (int kk = 0; kk < 2; ++kk)
                ax_mma_ts<F8>(TM_O, pa + c * 32 + kk * 8,
                              vb + (X::PU == 2 ? 0 : (c >> 1) * (X::VBOX >> 4)) + ((c & 1) * 2 + kk) * 2, id_hi, (i | c | kk) != 0);
            }
            if (unit_end) tc_commit(&vempty[v_st]);
            if (c == 3) {
              tc_commit(&pvdone[b]);
              if (i == n - 1) mbar_arrive(&iempty[it % AX_ITEMS]);
            }
          }
          __syncwarp();
          if (unit_end && ++v_st == X::NV) {
            v_st = 0;
            v_ph ^= 1;
          }
        }
        if (++b == X::NS) {
          b = 0;
          b_ph ^= 1;
        }
        if (ok) issue_s();
      }
      ++it;
    }
    if (*abort_flag) {   // let the MMAs in flight finish before the accumulators are given back
      const unsigned long long t0 = globaltimer();
      while (globaltimer() - t0 < 1000ull * 1000) {
      }
    }
  } else {
    // ---------------- softmax: TMEM quadrant q holds rows 32 q .., a lane owns a row.  Warp 4 + q takes the even pages and
    // warp 8 + q the odd ones (they share a scheduler: while one reads scores and looks for their maximum the other keeps
    // the exponential unit busy), and the running maximum passes between them ahead of the exponentials.  The probabilities
    // of 32 keys go where their scores were, and to the MMA issuer quarter by quarter ----------------
    const int q = warp & 3, e = (warp - AX_SOFT0) >> 2;
    const int row = q * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    const float sl2 = p.scale_log2;
    const int r_tok = row / p.grp, r_head = row - r_tok * p.grp;
    AxItem x;
    int tp0 = 0;                     // pages of the items before
    uint32_t pub = 0;                // maxima published by the other warp of the quadrant
    uint32_t ep = 0;                 // items of this quadrant
    bool ok = true;
    for (int it = 0; ok && item_wait(it, x); ++it) {
      const int n = x.p1 - x.p0;
      const bool active = q * 32 < x.ntok * p.grp;   // warps without a row only take part in the hand-overs
      const int lim = x.pos0 + r_tok;                // last key that this row sees
      const int32_t* tab = p.table + static_cast<size_t>(x.req) * p.pt_stride;
      if (p.gate && x.slot < 0 && r_tok < x.ntok && x.tok0 + r_tok < p.T) {   // the epilogue's gate rows, on their way to L2
        const bf16* g = p.gate + (x.tok0 + r_tok) * p.gate_stride + (x.head * p.grp + r_head) * D + e * (D / 2);
#pragma unroll
        for (int c = 0; c < D / 128; ++c) asm volatile("prefetch.global.L2 [%0];" ::"l"(g + c * 64));
      }
      float m_own = -INFINITY, l = 0.f;              // the maximum that l is relative to
      uint32_t bad = 0;                              // missing pages among 32
      for (int i = (tp0 & 1) ^ e; ok && i < n; i += 2) {
        const int tp = tp0 + i, pg = x.p0 + i, sb = tp % X::NS;
        const uint32_t sc = TM_S + sb * 128 + lanes;
        if (!active) {
          ok = ax_wait(&sfull[sb], (tp / X::NS) & 1, abort_flag, p.status, ST_WAIT_TMEM_FULL);
          if (ok && lane < 4) mbar_arrive(&pready[sb * 4 + lane]);
          continue;
        }
        if ((i & 31) < 2) {
          const int j = pg - (i & 31) + lane;
          const int id = j < x.p1 && j < p.pt_stride ? tab[j] : -1;
          bad = __ballot_sync(FULL_MASK, j < x.p1 && (id < 0 || id >= p.num_pages));
        }
        const bool gone = (bad >> (i & 31)) & 1;
        const bool edge = gone || pg * AX_PAGE + AX_PAGE - 1 > x.pos0;   // not every row sees all of the page
        const int see = gone ? -1 : lim - pg * AX_PAGE;
        ok = ax_wait(&sfull[sb], (tp / X::NS) & 1, abort_flag, p.status, ST_WAIT_TMEM_FULL);
        if (!ok) break;
        tc_fence_after();
        // the loops over a row's scores stay rolled: unrolled, a page's code overran the instruction cache, and the warps
        // waited for instructions a quarter of the time
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          uint32_t v[32];
          tmem_ld32(sc + c, v);
          tmem_ld_wait();
          if (edge) {                                // masked in place, so that the second pass need not ask
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j > see) v[j] = 0xff800000u;
            ax_tmem_st16(sc + c, v);
            ax_tmem_st16(sc + c + 16, v + 16);
          }
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
#pragma unroll
            for (int k = 0; k < 4; ++k) mx[k] = ax_max3(mx[k], __uint_as_float(v[j + k]), __uint_as_float(v[j + 4 + k]));
          }
        }
        if (edge) ax_tmem_st_wait();
        const float tm = fmaxf(ax_max3(mx[0], mx[1], mx[2]), mx[3]);
        // the maximum so far, of the page before
        float m = -INFINITY;
        if (i > 0) {
          ok = ax_wait(&mpub[(e ^ 1) * 4 + q], (pub + ((i + 1) >> 1) - 1) & 1, abort_flag, p.status, ST_WAIT_STATE);
          if (!ok) break;
          m = s_m[(e ^ 1) * 128 + row];
        }
        const bool move = (tm - m) * sl2 > AX_TAU;   // m = -inf: any finite maximum; both -inf: NaN, no move
        const float m_new = move ? tm : m;
        s_m[e * 128 + row] = m_new;
        __syncwarp();
        if (lane == 0) mbar_arrive(&mpub[e * 4 + q]);
        if (__any_sync(FULL_MASK, m_new != m_own)) {
          if (m_new != m_own) l *= ax_exp2((m_own - m_new) * sl2);
          m_own = m_new;
          if (i > 0 && __any_sync(FULL_MASK, move)) {
            // P . V of the page before.  Its barrier's phase before is known to be over (the scores of page tp came after
            // P . V of page tp - NS) and its next one cannot be (it needs this page), so the parity is not mistaken
            const float alpha = move ? ax_exp2((m - m_new) * sl2) : 1.f;
            ok = ax_wait(&pvdone[(tp - 1) % X::NS], ((tp - 1) / X::NS) & 1, abort_flag, p.status, ST_WAIT_TMEM_EMPTY);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t v[16];
              const uint32_t col = TM_O + c * 16 + lanes;
              tmem_ld16(col, v);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * alpha);
              ax_tmem_st16(col, v);
            }
          }
        }
        // rows of no token get zero probabilities (see the Q boxes)
        const float shift = r_tok < x.ntok ? (F8 ? AX_BIAS : 0.f) - (m_new == -INFINITY ? 0.f : m_new * sl2) : -INFINITY;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld32(sc + c * 32, v);
          tmem_ld_wait();
          uint32_t w[16];
          if (F8) {     // words 0..7: the values; 8..15: the remainders
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              float f[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(v[k * 4 + j]);
              ax_fma2(f[0], f[1], sl2, shift);
              ax_fma2(f[2], f[3], sl2, shift);
#pragma unroll
              for (int j = 0; j < 4; ++j) f[j] = ax_exp2(f[j]);
              ax_add2(acc[0], acc[1], f[0], f[1]);
              ax_add2(acc[2], acc[3], f[2], f[3]);
              const uint32_t f0 = ax_f16x2(f[0], f[1]), f1 = ax_f16x2(f[2], f[3]);
              const uint32_t h0 = ax_head(f0), h1 = ax_head(f1);
              w[k] = __byte_perm(h0, h1, 0x7531);
              w[8 + k] = ax_rest(f0, h0) | (ax_rest(f1, h1) << 16);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float f0 = __uint_as_float(v[k * 2]), f1 = __uint_as_float(v[k * 2 + 1]);
              ax_fma2(f0, f1, sl2, shift);
              w[k] = pack_bf2(ax_exp2(f0), ax_exp2(f1));
              ax_add2(acc[(k & 1) * 2], acc[(k & 1) * 2 + 1], bf_lo(w[k]), bf_hi(w[k]));   // the row sum takes the rounded
            }                                                                              // values: a common error cancels
          }
          ax_tmem_st16(sc + c * 32, w);
          ax_tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pready[sb * 4 + c]);
        }
        l += (acc[0] + acc[1]) + (acc[2] + acc[3]);
      }
      if (!ok) break;
      // ---- epilogue: the row sums of the two warps meet, each writes half of the columns of its rows ----
      const int last = tp0 + n - 1;                  // the last page; its warp knows when its P . V is done
      const bool mine = (last & 1) == e;
      const long long tok = x.tok0 + r_tok;
      const bool store = r_tok < x.ntok && tok < p.T;
      const int col0 = e * (D / 2);
      uint4 gv[4];
      const bool gated = p.gate && store && x.slot < 0;
      const uint4* g = reinterpret_cast<const uint4*>(p.gate + (gated ? tok * p.gate_stride + (x.head * p.grp + r_head) * D + col0 : 0));
      if (gated) {                                   // the first columns' gate, requested before the last P . V is waited for
#pragma unroll
        for (int j = 0; j < 4; ++j) gv[j] = g[j];
      }
      if (mine) ok = ax_wait(&pvdone[last % X::NS], (last / X::NS) & 1, abort_flag, p.status, ST_WAIT_TMEM_FULL);
      if (!ok) break;
      if (active) {
        pub += (n + ((tp0 & 1) ^ e)) >> 1;           // the other warp's pages: the larger half if it had the first
        float m = m_own;
        if (!mine) {
          ok = ax_wait(&mpub[(e ^ 1) * 4 + q], (pub - 1) & 1, abort_flag, p.status, ST_WAIT_STATE);
          if (!ok) break;
          m = s_m[(e ^ 1) * 128 + row];
          if (m_own != m) l *= ax_exp2((m_own - m) * sl2);
        }
        s_l[e * 128 + row] = l;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&lpub[q]);
        ok = ax_wait(&lpub[q], ep & 1, abort_flag, p.status, ST_WAIT_STATE);
        ++ep;
        if (!ok) break;
        tc_fence_after();
        const float total = l + s_l[(e ^ 1) * 128 + row];
        const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
        if (x.slot >= 0) {                           // partial: [column / 4][row], a warp's rows side by side
          float4* po = reinterpret_cast<float4*>(p.part) + (static_cast<size_t>(x.slot) * (D / 4) + col0 / 4) * p.rows + row;
#pragma unroll 1
          for (int c = 0; c < D / 64; ++c) {
            uint32_t v[32];
            tmem_ld32(TM_O + col0 + c * 32 + lanes, v);
            tmem_ld_wait();
            if (store) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                po[static_cast<size_t>(c * 8 + j) * p.rows] =
                    make_float4(__uint_as_float(v[j * 4]), __uint_as_float(v[j * 4 + 1]), __uint_as_float(v[j * 4 + 2]),
                                __uint_as_float(v[j * 4 + 3]));
            }
            __syncwarp();
          }
        } else {
          bf16* o = p.out + (tok * p.hq + x.head * p.grp + r_head) * D + col0;
#pragma unroll 1
          for (int c = 0; c < D / 64; ++c) {
            uint32_t v[32];
            tmem_ld32(TM_O + col0 + c * 32 + lanes, v);
            uint4 gc[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) gc[j] = gv[j];
            if (gated && c + 1 < D / 64) {           // the next columns' gate
#pragma unroll
              for (int j = 0; j < 4; ++j) gv[j] = g[(c + 1) * 4 + j];
            }
            tmem_ld_wait();
            if (store) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float f[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(v[j * 8 + k]) * inv;
                if (p.gate) {
                  const uint32_t gw[4] = {gc[j].x, gc[j].y, gc[j].z, gc[j].w};
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    f[k * 2] = __fdividef(f[k * 2], 1.f + __expf(-bf_lo(gw[k])));
                    f[k * 2 + 1] = __fdividef(f[k * 2 + 1], 1.f + __expf(-bf_hi(gw[k])));
                  }
                }
                reinterpret_cast<uint4*>(o + c * 32)[j] =
                    make_uint4(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]), pack_bf2(f[6], f[7]));
              }
            }
            __syncwarp();
          }
        }
        if (s_odd[it % AX_ITEMS] && store) ax_give_back<F8, D>(p, x, row, lim, tok, x.head * p.grp + r_head, col0);
        if (x.slot >= 0 && store && e == 0) {
          float* ml = p.part + static_cast<size_t>(2 * grid) * p.rows * D + static_cast<size_t>(x.slot) * 2 * p.rows;
          ml[row] = m * sl2;
          ml[p.rows + row] = total;
        }
        tc_fence_before();
      }
      tp0 += n;
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&ofree[it % AX_ITEMS]);
        mbar_arrive(&iempty[it % AX_ITEMS]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Merge of the tiles whose pages were cut: the pieces are added in page order with weights 2^(m - M), M the largest of their
// maxima.  One CTA per (range that a cut tile's second piece belongs to, 32 rows, 128 columns); a lane owns a row, a warp 16 of
// the columns.  Where a tile has 8 or 16 rows (decode, where a long history is cut into many pieces) the lanes' groups share
// the pieces between them and add up at the end, always in the same order.
constexpr int AX_MAX_PIECES = 160;
template <int D>
__global__ void __launch_bounds__(256, 4) attn_extend_merge_kernel(const AxArgs p, int grid) {
  __shared__ float s_m[AX_MAX_PIECES][32];
  pdl_wait();
  pdl_launch();
  const int32_t* d = p.desc + blockIdx.x * 8;
  const int pieces = min(d[0], AX_MAX_PIECES);
  if (pieces <= 0) return;
  const int tok0 = d[1], ntok = d[2], head = d[3];
  const int row0 = blockIdx.y * 32, left = ntok * p.grp - row0;        // rows of the tile from row0 on
  if (left <= 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int span = left <= 8 ? 8 : left <= 16 ? 16 : 32;               // lanes per group
  const int sub = lane / span, subs = 32 / span, r = lane % span, row = row0 + r;
  const int tok = tok0 + row / p.grp;
  const bool live = r < left && tok < p.T;
  const int first = 2 * (static_cast<int>(blockIdx.x) - 1) + 1;        // then 2 * blockIdx.x, 2 * (blockIdx.x + 1), ...
  auto slot = [&](int i) -> size_t { return i == 0 ? first : 2 * (blockIdx.x + i - 1); };
  const float* ml = p.part + static_cast<size_t>(2 * grid) * p.rows * D;
  constexpr int V = 4;           // float4s of a warp's columns
  const int hd = head * p.grp + row % p.grp, col = blockIdx.z * 128 + warp * V * 4;
  uint2 gv[V];
  if (p.gate && live && sub == 0) {   // requested ahead of the partials
    const uint2* g = reinterpret_cast<const uint2*>(p.gate + tok * p.gate_stride + static_cast<long long>(hd) * D + col);
#pragma unroll
    for (int c = 0; c < V; ++c) gv[c] = g[c];
  }
  for (int i = warp * subs + sub; i < pieces; i += 8 * subs) s_m[i][r] = live ? ml[slot(i) * 2 * p.rows + row] : -INFINITY;
  __syncthreads();
  float M = -INFINITY;
  for (int i = sub; i < pieces; i += subs) M = fmaxf(M, s_m[i][r]);
  for (int o = span; o < 32; o <<= 1) M = fmaxf(M, __shfl_xor_sync(FULL_MASK, M, o));
  float4 acc[V] = {};
  float L = 0.f;
  const float4* part = reinterpret_cast<const float4*>(p.part) + static_cast<size_t>(col / 4) * p.rows + row;
#pragma unroll 2
  for (int i = sub; i < pieces; i += subs) {
    const float m = s_m[i][r], w = m == -INFINITY ? 0.f : ax_exp2(m - M);
    L = fmaf(live ? ml[slot(i) * 2 * p.rows + p.rows + row] : 0.f, w, L);
    const float4* x = part + slot(i) * (D / 4) * p.rows;
    float4 v[V];
#pragma unroll
    for (int c = 0; c < V; ++c) v[c] = live ? x[static_cast<size_t>(c) * p.rows] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      acc[c].x = fmaf(v[c].x, w, acc[c].x);
      acc[c].y = fmaf(v[c].y, w, acc[c].y);
      acc[c].z = fmaf(v[c].z, w, acc[c].z);
      acc[c].w = fmaf(v[c].w, w, acc[c].w);
    }
  }
  for (int o = span; o < 32; o <<= 1) {
    L += __shfl_xor_sync(FULL_MASK, L, o);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      acc[c].x += __shfl_xor_sync(FULL_MASK, acc[c].x, o);
      acc[c].y += __shfl_xor_sync(FULL_MASK, acc[c].y, o);
      acc[c].z += __shfl_xor_sync(FULL_MASK, acc[c].z, o);
      acc[c].w += __shfl_xor_sync(FULL_MASK, acc[c].w, o);
    }
  }
  if (!live || sub != 0) return;
  const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
  uint2* o = reinterpret_cast<uint2*>(p.out + (static_cast<long long>(tok) * p.hq + hd) * D + col);
#pragma unroll
  for (int c = 0; c < V; ++c) {
    float f[4] = {acc[c].x * inv, acc[c].y * inv, acc[c].z * inv, acc[c].w * inv};
    if (p.gate) {
      f[0] = __fdividef(f[0], 1.f + __expf(-bf_lo(gv[c].x)));
      f[1] = __fdividef(f[1], 1.f + __expf(-bf_hi(gv[c].x)));
      f[2] = __fdividef(f[2], 1.f + __expf(-bf_lo(gv[c].y)));
      f[3] = __fdividef(f[3], 1.f + __expf(-bf_hi(gv[c].y)));
    }
    o[c] = make_uint2(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]));
  }
}

static int ax_grid() { return sm_count() < AX_MAX_PIECES ? sm_count() : AX_MAX_PIECES; }

template <bool F8, int D>
static void ax_launch(const CUtensorMap& tmQ, const CUtensorMap& tmQs, const CUtensorMap& tmK, const CUtensorMap& tmV, const AxArgs& a, cudaStream_t st) {
  using X = AxShape<F8, D>;
  static DeviceOnce once;
  once.run([] { cudaFuncSetAttribute(attn_extend_kernel<F8, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, X::SMEM); });
  const int grid = ax_grid();
  launch_k(attn_extend_kernel<F8, D>, dim3(grid), dim3(AX_THREADS), X::SMEM, st, tmQ, tmQs, tmK, tmV, a);
  launch_k(attn_extend_merge_kernel<D>, dim3(grid, (a.rows + 31) / 32, D / 128), dim3(256), 0, st, a, grid);
}

// rows of a tile: the group's heads of as many tokens as fit 128 rows, or of all T
static int ax_tokens_per_tile(int T, int grp) {
  const int tpt = 128 / grp;
  return T < tpt ? T : tpt;
}

}  // namespace b200

using namespace b200;

extern "C" size_t b200_attn_extend_workspace_bytes(int T, int Hq, int Hkv, int D) {
  if (T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || Hq % Hkv || Hq / Hkv > 128) return 0;
  const size_t rows = static_cast<size_t>(ax_tokens_per_tile(T, Hq / Hkv)) * (Hq / Hkv), grid = ax_grid();
  return grid * 32 + 2 * grid * rows * (static_cast<size_t>(D) + 2) * 4;
}

extern "C" int b200_attn_extend(const void* q, long long q_stride, const void* gate, long long gate_stride,
                                const void* kcache, const void* vcache, int num_pages, const int32_t* page_table,
                                int pt_stride, const int32_t* cu_seqlens, const int32_t* seqlens, int B, int T, int Hq,
                                int Hkv, int D, int cache_bf16, float scale, void* out, void* ws, size_t ws_bytes,
                                int32_t* status, void* stream) {
  if (!q || !kcache || !vcache || !page_table || !cu_seqlens || !seqlens || !out || !ws)
    return fail(B200_E_ARG, "b200_attn_extend: null pointer");
  if (B <= 0 || B > 8192 || T <= 0 || T > (1 << 24) || num_pages <= 0 || pt_stride <= 0 || pt_stride > (1 << 23))
    return fail(B200_E_ARG, "b200_attn_extend: need 1 <= B <= 8192, 1 <= T <= 2^24, num_pages >= 1 and 1 <= pt_stride <= 2^23 "
                "(B=%d T=%d)", B, T);
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > 128 || Hkv > 128 || (D != 128 && D != 256))
    return fail(B200_E_ARG, "b200_attn_extend: need Hq a multiple of Hkv, at most 128 heads per group, D 128 or 256 "
                "(Hq=%d Hkv=%d D=%d)", Hq, Hkv, D);
  if (static_cast<long long>(num_pages) * Hkv * D > 0x7fffff00ll)
    return fail(B200_E_ARG, "b200_attn_extend: num_pages * Hkv * D must stay below 2^31 (%d pages)", num_pages);
  if (!(scale > 0.f) || !(scale < 1e30f)) return fail(B200_E_ARG, "b200_attn_extend: scale must be positive and finite");
  const long long row = static_cast<long long>(Hq) * D, es = cache_bf16 ? 2 : 1;
  if (q_stride < row || (gate && gate_stride < row))
    return fail(B200_E_ARG, "b200_attn_extend: a token stride is shorter than a token's row");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(gate) | reinterpret_cast<uintptr_t>(kcache) |
       reinterpret_cast<uintptr_t>(vcache) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(ws) |
       static_cast<uintptr_t>(q_stride * es) | static_cast<uintptr_t>(gate ? gate_stride * 2 : 0)) & 15)
    return fail(B200_E_ALIGN, "b200_attn_extend: tensors, token strides and workspace must be 16-byte aligned");
  if (ws_bytes < b200_attn_extend_workspace_bytes(T, Hq, Hkv, D))
    return fail(B200_E_WS, "b200_attn_extend: workspace %zu < %zu bytes", ws_bytes,
                b200_attn_extend_workspace_bytes(T, Hq, Hkv, D));
  CUtensorMap tmQ, tmQs, tmK, tmV;
  int rc;
  AxArgs a{};
  a.grp = Hq / Hkv;
  a.tpt = ax_tokens_per_tile(T, a.grp);
  a.rows = a.tpt * a.grp;
  if ((rc = make_tmap_bytes_3d(&tmQ, q, static_cast<uint64_t>(D) * es, Hq, T, static_cast<uint64_t>(D) * es,
                               static_cast<uint64_t>(q_stride) * es, a.grp, a.tpt, "q")))
    return rc;
  a.sub = a.grp % 8 == 0 ? 1 : a.grp % 4 == 0 ? 2 : a.grp % 2 == 0 ? 4 : 8;
  if (a.sub > a.tpt) a.sub = a.tpt;   // never used then: two such boxes do not fit the tile
  if ((rc = make_tmap_bytes_3d(&tmQs, q, static_cast<uint64_t>(D) * es, Hq, T, static_cast<uint64_t>(D) * es,
                               static_cast<uint64_t>(q_stride) * es, a.grp, a.sub, "q")))
    return rc;
  if ((rc = make_tmap_bytes_2d(&tmK, kcache, static_cast<uint64_t>(num_pages) * Hkv * AX_PAGE, static_cast<uint64_t>(D) * es,
                               AX_PAGE, "k cache")))
    return rc;
  if ((rc = make_tmap_bytes_2d(&tmV, vcache, static_cast<uint64_t>(num_pages) * Hkv * D, AX_PAGE * es, D, "v cache"))) return rc;
  a.gate = static_cast<const bf16*>(gate);
  a.gate_stride = gate_stride;
  a.vc = vcache;
  a.num_pages = num_pages;
  a.table = page_table;
  a.pt_stride = pt_stride;
  a.cu = cu_seqlens;
  a.seqlens = seqlens;
  a.B = B;
  a.T = T;
  a.hq = Hq;
  a.hkv = Hkv;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = static_cast<bf16*>(out);
  a.desc = static_cast<int32_t*>(ws);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + static_cast<size_t>(ax_grid()) * 32);
  a.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cache_bf16)
    D == 256 ? ax_launch<false, 256>(tmQ, tmQs, tmK, tmV, a, st) : ax_launch<false, 128>(tmQ, tmQs, tmK, tmV, a, st);
  else
    D == 256 ? ax_launch<true, 256>(tmQ, tmQs, tmK, tmV, a, st) : ax_launch<true, 128>(tmQ, tmQs, tmK, tmV, a, st);
  return launch_status("b200_attn_extend");
}
