// Attention of ragged chunks of new tokens over the paged KV cache (prompts in chunks, plain decode, mixed batches).
#include "common.cuh"
#include "host.h"

namespace b200 {

B200_DEFINE_WAIT_BUDGET_SETTER(set_wait_budget_attn_extend)

constexpr int AX_PAGE = 128;

struct AxArgs {
  const void* q;
  long long q_stride;
  const bf16* gate;
  long long gate_stride;
  const void* kc;
  const void* vc;
  int num_pages;
  const int32_t* table;
  int pt_stride;
  const int32_t* cu;
  const int32_t* seqlens;
  int B, T, hq, hkv;
  float scale_log2;
  bf16* out;
  int32_t* status;
};

__device__ __forceinline__ float ax_float(uint8_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(v)));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(r & 0xffffu)));
}
__device__ __forceinline__ float ax_float(bf16 v) { return bf2f(v); }

// One CTA per (token, kv head); heads of the group in slices of 8.
template <typename E, int D>
__global__ void __launch_bounds__(256) attn_extend_rows_kernel(const AxArgs p) {
  __shared__ float s_q[8][D], s_p[8][AX_PAGE], s_a[8], s_l[8];
  __shared__ int s_b;
  pdl_wait();
  pdl_launch();
  const int t = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv, grp = p.hq / p.hkv;
  if (threadIdx.x == 0) s_b = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < p.B; b += 256)
    if (p.cu[b] <= t && t < p.cu[b + 1]) s_b = b;
  __syncthreads();
  const int b = s_b;
  if (b < 0) return;
  const int n = p.seqlens[b] - (p.cu[b + 1] - p.cu[b]) + (t - p.cu[b]) + 1;   // keys that this token sees
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const E* kc = static_cast<const E*>(p.kc);
  const E* vc = static_cast<const E*>(p.vc);
  for (int g0 = 0; g0 < grp; g0 += 8) {
    const int ng = min(8, grp - g0);
    for (int i = threadIdx.x; i < ng * D; i += 256)
      s_q[i / D][i % D] = ax_float(static_cast<const E*>(p.q)[t * p.q_stride + (h * grp + g0 + i / D) * D + i % D]) * p.scale_log2;
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;   // m, l: head `warp`, in every lane
    for (int k0 = 0; k0 < n; k0 += AX_PAGE) {
      const int j = k0 / AX_PAGE;
      const int page = j < p.pt_stride ? p.table[static_cast<size_t>(b) * p.pt_stride + j] : -1;
      if (page < 0 || page >= p.num_pages) {
        if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, B200_ST_BAD_PAGE);
        continue;
      }
      __syncthreads();
      const size_t ph = static_cast<size_t>(page) * p.hkv + h;
      for (int key = warp; key < AX_PAGE; key += 8) {
        float acc[8] = {};
        for (int d = lane; d < D; d += 32) {
          const float kv = ax_float(kc[(ph * AX_PAGE + key) * D + d]);
#pragma unroll
          for (int g = 0; g < 8; ++g)
            if (g < ng) acc[g] = fmaf(kv, s_q[g][d], acc[g]);
        }
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          for (int x = 16; x > 0; x >>= 1) acc[g] += __shfl_xor_sync(FULL_MASK, acc[g], x);
          if (lane == g) s_p[g][key] = k0 + key < n ? acc[g] : -INFINITY;
        }
      }
      __syncthreads();
      if (warp < ng) {
        float mx = m;
        for (int c = lane; c < AX_PAGE; c += 32) mx = fmaxf(mx, s_p[warp][c]);
        for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL_MASK, mx, x));
        const float a = exp2f(m - mx);
        float s = 0.f;
        for (int c = lane; c < AX_PAGE; c += 32) {
          const float e = exp2f(s_p[warp][c] - mx);
          s_p[warp][c] = e;
          s += e;
        }
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(FULL_MASK, s, x);
        l = l * a + s;
        m = mx;
        if (lane == 0) s_a[warp] = a;
      }
      __syncthreads();
      if (threadIdx.x < D) {
        const int d = threadIdx.x;
#pragma unroll
        for (int g = 0; g < 8; ++g)
          if (g < ng) o[g] *= s_a[g];
        for (int c = 0; c < min(AX_PAGE, n - k0); ++c) {
          const float vv = ax_float(vc[(ph * D + d) * AX_PAGE + c]);
#pragma unroll
          for (int g = 0; g < 8; ++g)
            if (g < ng) o[g] = fmaf(s_p[g][c], vv, o[g]);
        }
      }
    }
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    if (threadIdx.x < D)
      for (int g = 0; g < ng; ++g) {
        const long long c = static_cast<long long>(h * grp + g0 + g) * D + threadIdx.x;
        float r = s_l[g] == 0.f ? 0.f : o[g] / s_l[g];
        if (p.gate) r = r / (1.f + __expf(-bf2f(p.gate[t * p.gate_stride + c])));
        p.out[static_cast<long long>(t) * p.hq * D + c] = f2bf(r);
      }
    __syncthreads();
  }
}

}  // namespace b200

using namespace b200;

extern "C" size_t b200_attn_extend_workspace_bytes(int T, int Hq, int Hkv, int D) {
  if (T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0) return 0;
  return 16;
}

extern "C" int b200_attn_extend(const void* q, long long q_stride, const void* gate, long long gate_stride,
                                const void* kcache, const void* vcache, int num_pages, const int32_t* page_table,
                                int pt_stride, const int32_t* cu_seqlens, const int32_t* seqlens, int B, int T, int Hq,
                                int Hkv, int D, int cache_bf16, float scale, void* out, void* ws, size_t ws_bytes,
                                int32_t* status, void* stream) {
  if (!q || !kcache || !vcache || !page_table || !cu_seqlens || !seqlens || !out || !ws)
    return fail(B200_E_ARG, "b200_attn_extend: null pointer");
  if (B <= 0 || B > 8192 || T <= 0 || T > (1 << 24) || num_pages <= 0 || pt_stride <= 0)
    return fail(B200_E_ARG, "b200_attn_extend: need 1 <= B <= 8192, 1 <= T <= 2^24, num_pages and pt_stride >= 1 (B=%d T=%d)",
                B, T);
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > 128 || Hkv > 128 || (D != 128 && D != 256))
    return fail(B200_E_ARG, "b200_attn_extend: need Hq a multiple of Hkv, at most 128 heads per group, D 128 or 256 "
                "(Hq=%d Hkv=%d D=%d)", Hq, Hkv, D);
  if (static_cast<long long>(num_pages) * Hkv * D > 0x7fffffffll)
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
  const AxArgs a{q, q_stride, static_cast<const bf16*>(gate), gate_stride, kcache, vcache, num_pages, page_table, pt_stride,
                 cu_seqlens, seqlens, B, T, Hq, Hkv, scale * 1.4426950408889634f, static_cast<bf16*>(out), status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(T * Hkv);
  if (cache_bf16) {
    if (D == 256) launch_k(attn_extend_rows_kernel<bf16, 256>, grid, dim3(256), 0, st, a);
    else launch_k(attn_extend_rows_kernel<bf16, 128>, grid, dim3(256), 0, st, a);
  } else {
    if (D == 256) launch_k(attn_extend_rows_kernel<uint8_t, 256>, grid, dim3(256), 0, st, a);
    else launch_k(attn_extend_rows_kernel<uint8_t, 128>, grid, dim3(256), 0, st, a);
  }
  return launch_status("b200_attn_extend");
}
