// Attention over the 4-bit paged cache, straight from the packed pages.
//
// O = sum_t p_t V_t with p = softmax(scale q.K_t), online (running maximum and
// sum in fp32), K and V = c*s + z per token and channel group.
// First form: one CTA per (row, query head, query token); each warp takes
// every fourth page, a lane a token of it for q.K, then a lane D/32 channels
// for P.V; the warps' partial results meet in shared memory.
#include "int4.cuh"

namespace akv {

struct Int4AttnParams {
  akv_int4_cache c;
  const int32_t* rows;
  const int32_t* n_new;
  int M, Hq;
  const uint16_t* q;
  int64_t q_sr, q_sh, q_sm;
  float scale;
  uint16_t* out;
  int64_t o_sr, o_sh, o_sm;
  float* lse;
  int* status;
};

constexpr int kAttnWarps = 4;

template <int D, bool BF>
__global__ void __launch_bounds__(kAttnWarps * 32) int4_attn_kernel(Int4AttnParams P) {
  constexpr int PER = D / 32;  // channels of a lane in P.V
  __shared__ float s_q[D];
  __shared__ float s_acc[kAttnWarps][D];
  __shared__ float s_m[kAttnWarps], s_l[kAttnWarps];
  const int m = blockIdx.x, hq = blockIdx.y, i = blockIdx.z;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const Int4Row row = int4_row(P.c, P.rows, P.n_new, i, P.M, P.status);
  const int group = P.c.group, G = D / group;
  const int h = hq / (P.Hq / P.c.kv_heads);
  const int see = row.seq >= 0 && m < row.n_new ? row.len - row.n_new + m + 1 : 0;  // tokens this query sees
  for (int d = t; d < D; d += kAttnWarps * 32)
    s_q[d] = elem_to_float<BF>(P.q[i * P.q_sr + hq * P.q_sh + m * P.q_sm + d]) * P.scale;
  __syncthreads();
  float mx = -INFINITY, l = 0.f, acc[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) acc[k] = 0.f;
  const int blocks = see > 0 ? (see + kBlockTokens - 1) / kBlockTokens : 0;
  for (int j = warp; j < blocks; j += kAttnWarps) {
    int page = P.c.table[row.seq * P.c.table_stride + j];
    if (page < 0 || page >= P.c.n_pages) {
      set_status(P.status, AKV_ERR_SHAPE);
      page = 0;
    }
    const uint8_t* rec = P.c.pool + page * P.c.page_stride + h * P.c.head_stride;
    const uint8_t* kr = rec + lane * (D / 2);
    const __half2* kp = reinterpret_cast<const __half2*>(rec + kBlockTokens * D) + lane * G;
    const __half2* vp = reinterpret_cast<const __half2*>(rec + kBlockTokens * D + kBlockTokens * G * 4);
    float x = 0.f;
    for (int g = 0; g < G; ++g) {
      const float ks = __low2float(kp[g]), kz = __high2float(kp[g]);
      for (int d = g * group; d < (g + 1) * group; d += 8) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(kr + d / 2);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x = fmaf(s_q[d + e], fmaf(static_cast<float>((w >> (8 * (e >> 1) + (e & 1 ? 0 : 4))) & 15u), ks, kz), x);
      }
    }
    if (j * kBlockTokens + lane >= see) x = -INFINITY;
    float top = x;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float m2 = fmaxf(mx, top);  // finite: a visited page holds a visible token
    const float r = expf(mx - m2), p = expf(x - m2);
    mx = m2;
    l = l * r + p;
#pragma unroll
    for (int k = 0; k < PER; ++k) acc[k] *= r;
    for (int s = 0; s < kBlockTokens; ++s) {
      const float ps = __shfl_sync(~0u, p, s);
      const int d0 = lane * PER;
      const __half2 sz = vp[s * G + d0 / group];
      const uint8_t* vr = rec + kBlockTokens * D / 2 + s * (D / 2) + d0 / 2;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const uint32_t c = (vr[k / 2] >> (k & 1 ? 0 : 4)) & 15u;
        if (ps != 0.f) acc[k] = fmaf(ps, fmaf(static_cast<float>(c), __low2float(sz), __high2float(sz)), acc[k]);
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
#pragma unroll
  for (int k = 0; k < PER; ++k) s_acc[warp][lane * PER + k] = acc[k];
  if (lane == 0) {
    s_m[warp] = mx;
    s_l[warp] = l;
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, s_m[w]);
  float f[kAttnWarps];
  for (int w = 0; w < kAttnWarps; ++w) {
    f[w] = s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - top);
    sum += f[w] * s_l[w];
  }
  for (int d = t; d < D; d += kAttnWarps * 32) {
    float o = 0.f;
    for (int w = 0; w < kAttnWarps; ++w) o += f[w] * s_acc[w][d];
    P.out[i * P.o_sr + hq * P.o_sh + m * P.o_sm + d] = float_to_elem<BF>(sum > 0.f ? o / sum : 0.f);
  }
  if (P.lse && t == 0)
    P.lse[(static_cast<int64_t>(i) * P.Hq + hq) * P.M + m] = sum > 0.f ? top + logf(sum) : -INFINITY;
}

}  // namespace akv

using namespace akv;

template <int D>
static void attn_launch(const Int4AttnParams& p, int R, bool bf, cudaStream_t st) {
  const dim3 grid(p.M, p.Hq, R);
  if (bf) int4_attn_kernel<D, true><<<grid, kAttnWarps * 32, 0, st>>>(p);
  else int4_attn_kernel<D, false><<<grid, kAttnWarps * 32, 0, st>>>(p);
}

extern "C" size_t akv_int4_attention_workspace_bytes(int R, int M, int Hq, int kv_heads, int head_dim, int max_blocks) {
  if (R < 0 || M < 0 || Hq <= 0 || kv_heads <= 0 || Hq % kv_heads || max_blocks <= 0) return 0;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
  return 16;
}

extern "C" int akv_int4_attention(const akv_int4_cache* c, const int32_t* rows, const int32_t* n_new, int R, int M,
                                  int Hq, const void* q, int64_t q_sr, int64_t q_sh, int64_t q_sm, float sm_scale,
                                  void* out, int64_t o_sr, int64_t o_sh, int64_t o_sm, float* lse, int dtype,
                                  void* workspace, size_t workspace_bytes, int* status, void* stream) {
  const int rc = int4_check(c);
  if (rc) return rc;
  if (dtype != AKV_FP16 && dtype != AKV_BF16) return AKV_ERR_UNSUPPORTED;
  if (R < 0 || M < 0 || Hq <= 0 || Hq % c->kv_heads) return AKV_ERR_SHAPE;
  if (R == 0 || M == 0) return AKV_OK;
  if (!q || !out || !workspace) return AKV_ERR_NULL;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 1) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15))
    return AKV_ERR_ALIGN;
  if (R > 65535 || Hq > 65535) return AKV_ERR_UNSUPPORTED;
  if (workspace_bytes < akv_int4_attention_workspace_bytes(R, M, Hq, c->kv_heads, c->head_dim, c->max_blocks))
    return AKV_ERR_WORKSPACE;
  const Int4AttnParams p{*c, rows, n_new, M, Hq, static_cast<const uint16_t*>(q), q_sr, q_sh, q_sm, sm_scale,
                         static_cast<uint16_t*>(out), o_sr, o_sh, o_sm, lse, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == AKV_BF16;
  if (c->head_dim == 64) attn_launch<64>(p, R, bf, st);
  else if (c->head_dim == 128) attn_launch<128>(p, R, bf, st);
  else attn_launch<256>(p, R, bf, st);
  return cudaGetLastError() == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH;
}
