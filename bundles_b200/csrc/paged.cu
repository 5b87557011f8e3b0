// The paged KV cache around the attention: block tables, positions and slot maps from request lengths
// (page_plan_kernel), and the writer of a ragged batch of new tokens' K and V into the pages (kv_append).
// No counterpart in the reference: its engine builds both on the host and hands the kernels a per-token table
// (qk_attn_verify.cu:398-423).
#include "common.cuh"
#include "host.h"

namespace b200 {

constexpr int PG_TOKENS = 128;     // tokens of a page
constexpr int PP_THREADS = 1024;
constexpr int PP_MAX_BATCH = 8192;

struct PlanArgs {
  const int32_t* ctx;
  const int32_t* fresh;     // new tokens per request
  int B;
  int32_t* table;           // [B, pt_stride]
  int pt_stride, num_pages;
  const int32_t* free_pages;
  int free_cap;
  const int32_t* n_free;
  int T;
  int32_t* cu;
  int32_t* seqlens;
  int64_t* positions;
  int64_t* slots;
  int32_t* n_left;
  int32_t* status;
};

__device__ __forceinline__ void flag(int32_t* status, int code) {
  if (status) atomicCAS(status, 0, code);
}

// Exclusive prefix sum over the CTA of one value per thread; `total` is the sum.  `tmp`: 33 words of shared memory.
__device__ __forceinline__ long long block_scan(long long v, long long* tmp, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(FULL_MASK, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) tmp[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    long long w = lane < nw ? tmp[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(FULL_MASK, w, o);
      if (lane >= o) w += u;
    }
    if (lane < nw) tmp[lane] = w;
  }
  __syncthreads();
  total = tmp[nw - 1];
  const long long before = (warp ? tmp[warp - 1] : 0) + inc - v;
  __syncthreads();
  return before;
}

// Last index b in [0, n) with a[b] <= x (a ascending, a[0] <= x).
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Every CTA forms the two prefix sums over the batch (first row and first new page of every request) in its own shared
// memory and then fills its share of the token rows and of the new table entries: the CTAs exchange nothing, so one
// launch does it all.  An entry that a token reads is either an old one, which nobody writes, or taken from the free
// list directly, which nobody writes either.  Bound: latency, of the launch, the loads of the lengths and two block scans; 3.5 us
// from one request to 1500 with 27 k tokens (the host side of the call takes 18).
__global__ void __launch_bounds__(PP_THREADS) page_plan_kernel(const PlanArgs p) {
  extern __shared__ int pp_smem[];
  __shared__ long long tmp[33];
  int* s_cu = pp_smem;                   // [B + 1] first row of a request
  int* s_pg = pp_smem + p.B + 1;         // [B + 1] first new page of a request, counted over the batch
  int* s_ctx = pp_smem + 2 * (p.B + 1);  // [B] tokens already cached
  pdl_wait();
  pdl_launch();
  const int tid = threadIdx.x;
  const bool first = blockIdx.x == 0;
  const int per = (p.B + PP_THREADS - 1) / PP_THREADS, b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
  const long long cap = static_cast<long long>(p.pt_stride) * PG_TOKENS;
  long long sum = 0, total;
  for (int b = b0; b < b1; ++b) {
    const int n = p.fresh[b], c = p.ctx[b];
    if (first && (n < 0 || c < 0)) flag(p.status, B200_ST_BAD_LEN);
    if (first && c > cap) flag(p.status, B200_ST_NO_PAGE);
    s_ctx[b] = static_cast<int>(min(static_cast<long long>(max(c, 0)), min(cap, 0x3fffffffll)));
    sum += max(n, 0);
  }
  long long at = block_scan(sum, tmp, total);
  if (first && tid == 0 && total > p.T) flag(p.status, B200_ST_BAD_LEN);
  for (int b = b0; b < b1; ++b) {
    s_cu[b] = static_cast<int>(min(at, static_cast<long long>(p.T)));
    at += max(p.fresh[b], 0);
  }
  if (tid == 0) s_cu[p.B] = static_cast<int>(min(total, static_cast<long long>(p.T)));
  __syncthreads();
  sum = 0;
  auto pages = [&](int b) -> int {   // new pages of request b inside the table
    const int have = (s_ctx[b] + PG_TOKENS - 1) / PG_TOKENS;
    const int need = (s_ctx[b] + (s_cu[b + 1] - s_cu[b]) + PG_TOKENS - 1) / PG_TOKENS;
    return max(0, min(need, p.pt_stride) - have);
  };
  for (int b = b0; b < b1; ++b) sum += pages(b);
  at = block_scan(sum, tmp, total);
  for (int b = b0; b < b1; ++b) {
    s_pg[b] = static_cast<int>(at);
    at += pages(b);
  }
  if (tid == 0) s_pg[p.B] = static_cast<int>(total);
  __syncthreads();
  const int n_new = s_pg[p.B], n_tok = s_cu[p.B];
  const int n_free = p.free_pages ? max(0, min(*p.n_free, p.free_cap)) : 0;
  if (first) {
    for (int b = tid; b <= p.B; b += PP_THREADS) {
      p.cu[b] = s_cu[b];
      if (b < p.B) p.seqlens[b] = s_ctx[b] + (s_cu[b + 1] - s_cu[b]);
    }
    if (tid == 0 && p.n_left) *p.n_left = max(0, n_free - n_new);
  }
  const int g0 = blockIdx.x * PP_THREADS + tid, gn = gridDim.x * PP_THREADS;
  // the k-th new page of the batch comes off the end of the free list
  auto taken = [&](int k) -> int {
    if (k >= n_free) return -1;
    const int id = p.free_pages[n_free - 1 - k];
    return id >= 0 && id < p.num_pages ? id : -2;
  };
  if (p.free_pages)
    for (int k = g0; k < n_new; k += gn) {
      const int b = last_not_above(s_pg, p.B + 1, k);
      const int id = taken(k);
      if (id < 0) flag(p.status, id == -1 ? B200_ST_NO_PAGE : B200_ST_BAD_PAGE);
      p.table[static_cast<size_t>(b) * p.pt_stride + (s_ctx[b] + PG_TOKENS - 1) / PG_TOKENS + (k - s_pg[b])] = max(id, -1);
    }
  for (int t = g0; t < p.T; t += gn) {
    long long pos = 0, slot = -1;
    if (t < n_tok) {
      const int b = last_not_above(s_cu, p.B + 1, t);
      pos = static_cast<long long>(s_ctx[b]) + (t - s_cu[b]);
      const int j = static_cast<int>(pos / PG_TOKENS), have = (s_ctx[b] + PG_TOKENS - 1) / PG_TOKENS;
      int id;
      if (j >= p.pt_stride) {
        id = -1;
      } else if (j < have || !p.free_pages) {
        id = p.table[static_cast<size_t>(b) * p.pt_stride + j];
        if (id < 0 || id >= p.num_pages) id = -2;
      } else {
        id = taken(s_pg[b] + j - have);
      }
      if (id >= 0)
        slot = static_cast<long long>(id) * PG_TOKENS + pos % PG_TOKENS;
      else
        flag(p.status, id == -1 ? B200_ST_NO_PAGE : B200_ST_BAD_PAGE);
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
}

// The append copies K rows as they are and turns V rows into columns of the dim-major pages.  A CTA takes KA_TOK tokens and 64 dims of
// one kv head: the tokens that fill 128 bytes of a page's V row, or 16 where that would leave most of the GPU idle (64
// decoded tokens: 8 CTAs, 7.6 us; 32 CTAs, 3.0 us).  The tokens are cut into pieces that share one aligned
// 16-byte chunk of a page (a new piece starts where the slots do not follow on, and at every chunk); eight neighbouring
// lanes take neighbouring pieces of the same dims, so whole pages are written in full 128-byte lines.  A piece that is not
// a whole chunk (a lone decoded token) is written element by element.  V passes through shared memory in 4-byte words
// whose place is rotated by the piece, so that the eight lanes read different banks.
// Bound: HBM for prompts; the two dependent loads (slot, row) and the launch for a decode step.
constexpr int KA_DIMS = 64, KA_THREADS = 128;

template <typename E, int KA_TOK>
__global__ void __launch_bounds__(KA_THREADS) kv_append_kernel(const E* __restrict__ k, const E* __restrict__ v,
                                                               long long k_stride, long long v_stride, int T, int hkv, int dim,
                                                               E* __restrict__ kc, E* __restrict__ vc, int num_pages,
                                                               const int64_t* __restrict__ slots, int32_t* status) {
  constexpr int ES = sizeof(E), G = 16 / ES;                       // tokens of a chunk
  constexpr int ROW_W = KA_DIMS * ES / 4, ROW_Q = KA_DIMS * ES / 16;   // words and 16-byte quarters of a token's slice
  constexpr int PER_W = 4 / ES;                                    // dims of a word
  __shared__ long long s_slot[KA_TOK];
  __shared__ int s_start[KA_TOK + 1];
  __shared__ int s_cnt[4];
  __shared__ __align__(16) uint32_t s_v[KA_TOK * ROW_W];
  pdl_wait();
  pdl_launch();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int slices = dim / KA_DIMS;
  const int d0 = (blockIdx.x % slices) * KA_DIMS, h = (blockIdx.x / slices) % hkv;
  const long long t0 = static_cast<long long>(blockIdx.x / slices / hkv) * KA_TOK;
  const int n = static_cast<int>(min(static_cast<long long>(KA_TOK), T - t0));
  long long slot = -1;
  if (tid < n) {
    slot = slots[t0 + tid];
    if (slot >= static_cast<long long>(num_pages) * PG_TOKENS) {
      flag(status, B200_ST_BAD_PAGE);
      slot = -1;
    }
    if (slot < 0) slot = -1;
  }
  if (tid < KA_TOK) s_slot[tid] = slot;
  // both tiles are requested before the slots are looked at
  constexpr int LD = (KA_TOK * ROW_Q + KA_THREADS - 1) / KA_THREADS;
  uint4 kr[LD], vr[LD];
#pragma unroll
  for (int i = 0; i < LD; ++i) {
    const int t = (tid + i * KA_THREADS) / ROW_Q, c = (tid + i * KA_THREADS) % ROW_Q;
    if (t < n) {
      kr[i] = *reinterpret_cast<const uint4*>(k + (t0 + t) * k_stride + static_cast<long long>(h) * dim + d0 + c * G);
      vr[i] = *reinterpret_cast<const uint4*>(v + (t0 + t) * v_stride + static_cast<long long>(h) * dim + d0 + c * G);
    }
  }
  __syncthreads();
  const bool start = tid < n && (tid == 0 || slot != s_slot[tid - 1] + 1 || slot % G == 0 || slot < 0);
  const unsigned ball = __ballot_sync(FULL_MASK, start);
  if (lane == 0) s_cnt[warp] = __popc(ball);
#pragma unroll
  for (int i = 0; i < LD; ++i) {
    const int t = (tid + i * KA_THREADS) / ROW_Q, c = (tid + i * KA_THREADS) % ROW_Q;
    if (t < n) {
      const long long sl = s_slot[t];
      if (sl >= 0) *reinterpret_cast<uint4*>(kc + ((sl / PG_TOKENS * hkv + h) * PG_TOKENS + sl % PG_TOKENS) * dim + d0 + c * G) = kr[i];
      // a token's words are rotated by 4 for every chunk's worth of tokens
      uint32_t* row = s_v + t * ROW_W;
      const int rot = (t / G) * 4;
      *reinterpret_cast<uint4*>(row + ((c * 4 + rot) & (ROW_W - 1))) = vr[i];
    }
  }
  __syncthreads();
  int before = 0, pieces = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < warp) before += s_cnt[w];
    pieces += s_cnt[w];
  }
  if (start) s_start[before + __popc(ball & ((1u << lane) - 1))] = tid;
  if (tid == 0) s_start[pieces] = n;
  __syncthreads();
  // items: 8 pieces x the words of a slice, pieces fastest
  const int items = (pieces + 7) / 8 * 8 * ROW_W;
  for (int it = tid; it < items; it += KA_THREADS) {
    const int pc = it / (8 * ROW_W) * 8 + (it & 7), wd = (it >> 3) % ROW_W;
    if (pc >= pieces) continue;
    const int a = s_start[pc], cnt = s_start[pc + 1] - a;
    const long long sl = s_slot[a];
    if (sl < 0) continue;
    E* dst = vc + ((sl / PG_TOKENS * hkv + h) * dim + d0 + wd * PER_W) * PG_TOKENS + sl % PG_TOKENS;
    auto word = [&](int t) -> uint32_t { return s_v[t * ROW_W + ((wd + (t / G) * 4) & (ROW_W - 1))]; };
    if (cnt == G) {
      uint32_t x[G];
#pragma unroll
      for (int j = 0; j < G; ++j) x[j] = word(a + j);
#pragma unroll
      for (int e = 0; e < PER_W; ++e) {   // dim e of the word: its elements of the G tokens, side by side
        uint32_t y[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (ES == 1) {
            const uint32_t lo = __byte_perm(x[q * 4], x[q * 4 + 1], e | ((4 + e) << 4));
            const uint32_t hi = __byte_perm(x[q * 4 + 2], x[q * 4 + 3], e | ((4 + e) << 4));
            y[q] = __byte_perm(lo, hi, 0x5410);
          } else {
            y[q] = __byte_perm(x[q * 2], x[q * 2 + 1], e ? 0x7632 : 0x5410);
          }
        }
        *reinterpret_cast<uint4*>(dst + e * PG_TOKENS) = make_uint4(y[0], y[1], y[2], y[3]);
      }
    } else {
      for (int j = 0; j < cnt; ++j) {
        const uint32_t x = word(a + j);
#pragma unroll
        for (int e = 0; e < PER_W; ++e) dst[e * PG_TOKENS + j] = static_cast<E>(x >> (e * 8 * ES));
      }
    }
  }
}

template <typename E, int WIDE>
static void ka_launch(bool narrow, unsigned grid, const void* k, const void* v, long long ks, long long vs, int T, int hkv, int dim,
                      void* kc, void* vc, int pages, const int64_t* slots, int32_t* status, cudaStream_t st) {
  launch_k(narrow ? kv_append_kernel<E, 16> : kv_append_kernel<E, WIDE>, dim3(grid), dim3(KA_THREADS), 0, st,
           static_cast<const E*>(k), static_cast<const E*>(v), ks, vs, T, hkv, dim, static_cast<E*>(kc), static_cast<E*>(vc), pages,
           slots, status);
}

}  // namespace b200

using namespace b200;

extern "C" int b200_page_plan(const int32_t* ctx_lens, const int32_t* new_lens, int B, int32_t* page_table, int pt_stride,
                              int num_pages, const int32_t* free_pages, int free_cap, const int32_t* n_free, int T,
                              int32_t* cu_seqlens, int32_t* seqlens, int64_t* positions, int64_t* slots, int32_t* n_left,
                              int32_t* status, void* stream) {
  if (!ctx_lens || !new_lens || !page_table || !cu_seqlens || !seqlens || !positions || !slots)
    return fail(B200_E_ARG, "b200_page_plan: null pointer");
  if (free_pages && (!n_free || !n_left)) return fail(B200_E_ARG, "b200_page_plan: a free list needs n_free and n_left");
  if (B <= 0 || B > PP_MAX_BATCH || T <= 0 || pt_stride <= 0 || num_pages <= 0 || (free_pages && free_cap <= 0))
    return fail(B200_E_ARG, "b200_page_plan: need 1 <= B <= %d, T, pt_stride, num_pages and free_cap >= 1 (B=%d T=%d)",
                PP_MAX_BATCH, B, T);
  if (pt_stride > (1 << 23) || T > (1 << 29)) return fail(B200_E_ARG, "b200_page_plan: pt_stride <= 2^23 and T <= 2^29");
  static DeviceOnce once;
  once.run([] {
    cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (3 * PP_MAX_BATCH + 2) * 4);
  });
  const PlanArgs a{ctx_lens, new_lens, B,  page_table, pt_stride, num_pages, free_pages, free_cap,
                   n_free,   T,        cu_seqlens, seqlens, positions, slots, n_left, status};
  int grid = (T + PP_THREADS - 1) / PP_THREADS;
  if (grid > sm_count()) grid = sm_count();
  launch_k(page_plan_kernel, dim3(grid), dim3(PP_THREADS), (3 * static_cast<size_t>(B) + 2) * 4,
           static_cast<cudaStream_t>(stream), a);
  return launch_status("b200_page_plan");
}

extern "C" int b200_kv_append(const void* k, const void* v, long long k_stride, long long v_stride, int T, int Hkv, int D,
                              int cache_bf16, void* kcache, void* vcache, int num_pages, const int64_t* slots,
                              int32_t* status, void* stream) {
  if (!k || !v || !kcache || !vcache || !slots) return fail(B200_E_ARG, "b200_kv_append: null pointer");
  if (T < 0 || Hkv <= 0 || Hkv > 128 || (D != 128 && D != 256) || num_pages <= 0)
    return fail(B200_E_ARG, "b200_kv_append: need T >= 0, 1 <= Hkv <= 128, D 128 or 256 and num_pages >= 1 (Hkv=%d D=%d)", Hkv,
                D);
  const long long es = cache_bf16 ? 2 : 1;
  if (k_stride < static_cast<long long>(Hkv) * D || v_stride < static_cast<long long>(Hkv) * D)
    return fail(B200_E_ARG, "b200_kv_append: a token stride is shorter than a token's row");
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(kcache) |
        reinterpret_cast<uintptr_t>(vcache) | static_cast<uintptr_t>(k_stride * es) | static_cast<uintptr_t>(v_stride * es)) & 15))
    return fail(B200_E_ALIGN, "b200_kv_append: tensors and token strides must be 16-byte aligned");
  if (T == 0) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long wide = cache_bf16 ? 64 : 128, cols = static_cast<long long>(Hkv) * (D / KA_DIMS);
  const bool narrow = (T + wide - 1) / wide * cols < sm_count() / 2;
  const long long grid = (narrow ? (T + 15) / 16 : (T + wide - 1) / wide) * cols;
  if (grid > 0x7fffffffll) return fail(B200_E_ARG, "b200_kv_append: too many tokens (T=%d)", T);
  if (cache_bf16)
    ka_launch<uint16_t, 64>(narrow, static_cast<unsigned>(grid), k, v, k_stride, v_stride, T, Hkv, D, kcache, vcache, num_pages,
                            slots, status, st);
  else
    ka_launch<uint8_t, 128>(narrow, static_cast<unsigned>(grid), k, v, k_stride, v_stride, T, Hkv, D, kcache, vcache, num_pages,
                            slots, status, st);
  return launch_status("b200_kv_append");
}
