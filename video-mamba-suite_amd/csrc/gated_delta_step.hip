// gated_delta_step.hip -- gated delta rule, one token (vms_gated_delta_state_update):
//   S' = exp(g) S;  u = beta (v - S'^T k);  S = S' + k u^T;  out = scale S^T q = scale (S'^T q + (k.q) u)
// The second form of `out` needs S' only, so one reduction over the rows (S'^T k, S'^T q, k.q together) and one pass over the state:
// a streaming kernel, bound by the state's bytes (read and written once).  A workgroup owns 32 columns of one head's state, a thread
// 4 columns (16 bytes of fp32) of every 32nd row, all of it in registers between the reduction and the store; rows of 128 bytes.
// Few columns per workgroup because one sequence has few heads: (1, 8 heads, 128 x 128) is 32 workgroups instead of 8.
#include "vms_common.h"

namespace vms {
namespace gds {

constexpr int kCols = 32, kGroups = 32;   // columns of a workgroup; row groups (8 per wave)

__device__ __forceinline__ float ld(const void* p, int64_t i, int dt) {
    if (dt == VMS_F32) return static_cast<const float*>(p)[i];
    if (dt == VMS_F16) return static_cast<float>(static_cast<const f16_t*>(p)[i]);
    return static_cast<float>(static_cast<const bf16_t*>(p)[i]);
}
template <typename TS>
__device__ __forceinline__ void ld4(const TS* p, int n, float (&o)[4]) {
    TS v[4] = {};
    if (n >= 4) __builtin_memcpy(v, p, sizeof(v));
    else
        for (int e = 0; e < 4; ++e)
            if (e < n) v[e] = p[e];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = static_cast<float>(v[e]);
}
template <typename TS>
__device__ __forceinline__ void st4(TS* p, int n, const float (&o)[4]) {
    TS v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<TS>(o[e]);
    if (n >= 4) __builtin_memcpy(p, v, sizeof(v));
    else
        for (int e = 0; e < 4; ++e)
            if (e < n) p[e] = v[e];
}

// TS: the state's type; RPT: rows of a thread (dk <= 32 RPT)
template <typename TS, int RPT>
__global__ __launch_bounds__(256) void gd_step_kernel(const vms_gated_delta_step_params p, const int slices) {
    __shared__ float red[4][8][12];   // [wave][column group][S'^T k x4, S'^T q x4, k.q]
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, cg = lane & 7, rg = w * 8 + (lane >> 3);
    const int slice = blockIdx.x % slices;
    const int64_t pair = blockIdx.x / slices;
    const int b = (int)(pair / p.heads), h = (int)(pair % p.heads), hk = h / (p.heads / p.heads_k);
    const int c0 = slice * kCols + 4 * cg, nc = p.dv - c0;   // nc <= 0: no column of this thread
    TS* const S = static_cast<TS*>(p.state) + (int64_t)b * p.state_batch_stride + (int64_t)h * p.state_head_stride;
    const int64_t qo = (int64_t)b * p.q_batch_stride + (int64_t)hk * p.q_head_stride, ko = (int64_t)b * p.k_batch_stride + (int64_t)hk * p.k_head_stride;
    float s[RPT][4], kv[RPT], qv[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int row = rg + kGroups * i;
        kv[i] = row < p.dk ? ld(p.k, ko + row, p.dtype) : 0.f;
        qv[i] = row < p.dk ? ld(p.q, qo + row, p.dtype) : 0.f;
        if (row < p.dk && nc > 0) ld4<TS>(S + (int64_t)row * p.dv + c0, nc, s[i]);
        else
            for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
    }
    const float a = fast_exp(ld(p.g, (int64_t)b * p.g_batch_stride + (int64_t)h * p.g_head_stride, p.gate_dtype));
    const float be = ld(p.beta, (int64_t)b * p.beta_batch_stride + (int64_t)h * p.beta_head_stride, p.gate_dtype);
    float x[9] = {};
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s[i][e] *= a;
            x[e] = fmaf(s[i][e], kv[i], x[e]);
            x[4 + e] = fmaf(s[i][e], qv[i], x[4 + e]);
        }
        x[8] = fmaf(kv[i], qv[i], x[8]);
    }
#pragma unroll
    for (int m = 8; m < 64; m *= 2)
#pragma unroll
        for (int e = 0; e < 9; ++e) x[e] += __shfl_xor(x[e], m);
    if (lane < 8)
#pragma unroll
        for (int e = 0; e < 9; ++e) red[w][cg][e] = x[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 9; ++e) x[e] = red[0][cg][e] + red[1][cg][e] + red[2][cg][e] + red[3][cg][e];
    if (nc <= 0) return;
    float u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float v = e < nc ? ld(p.v, (int64_t)b * p.v_batch_stride + (int64_t)h * p.v_head_stride + c0 + e, p.dtype) : 0.f;
        u[e] = be * (v - x[e]);
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int row = rg + kGroups * i;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = fmaf(kv[i], u[e], s[i][e]);
        if (row < p.dk) st4<TS>(S + (int64_t)row * p.dv + c0, nc, s[i]);
    }
    if (rg == 0) {
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = p.scale * fmaf(x[8], u[e], x[4 + e]);
        const int64_t at = (int64_t)b * p.out_batch_stride + (int64_t)h * p.out_head_stride + c0;
        if (p.dtype == VMS_F32) st4<float>(static_cast<float*>(p.out) + at, nc, o);
        else if (p.dtype == VMS_F16) st4<f16_t>(static_cast<f16_t*>(p.out) + at, nc, o);
        else st4<bf16_t>(static_cast<bf16_t*>(p.out) + at, nc, o);
    }
}

template <typename TS>
static void launch(const vms_gated_delta_step_params& p, hipStream_t s) {
    const int slices = (p.dv + kCols - 1) / kCols;
    const dim3 grid((unsigned)((int64_t)p.batch * p.heads * slices)), block(256);
    if (p.dk <= 32) hipLaunchKernelGGL((gd_step_kernel<TS, 1>), grid, block, 0, s, p, slices);
    else if (p.dk <= 64) hipLaunchKernelGGL((gd_step_kernel<TS, 2>), grid, block, 0, s, p, slices);
    else hipLaunchKernelGGL((gd_step_kernel<TS, 4>), grid, block, 0, s, p, slices);
}

}  // namespace gds
}  // namespace vms

using namespace vms;

extern "C" int vms_gated_delta_state_update(const vms_gated_delta_step_params* pp, void* stream) {
    VMS_CHECK(pp != nullptr, "null params");
    const vms_gated_delta_step_params& p = *pp;
    auto dt_ok = [](int d) { return d == VMS_F32 || d == VMS_F16 || d == VMS_BF16; };
    VMS_CHECK(dt_ok(p.state_dtype) && dt_ok(p.dtype), "dtypes must be fp32/fp16/bf16");
    VMS_CHECK(p.gate_dtype == VMS_F32 || p.gate_dtype == p.dtype, "g and beta must be fp32 or of the activations' type");
    VMS_CHECK(p.batch > 0 && p.heads > 0 && p.heads_k > 0, "empty problem");
    VMS_CHECK(p.heads % p.heads_k == 0, "heads must be a multiple of heads_k");
    VMS_CHECK(p.dk >= 1 && p.dk <= 128 && p.dv >= 1 && p.dv <= 4096, "key heads of 1 .. 128, value heads of 1 .. 4096");
    VMS_CHECK((int64_t)p.batch * p.heads * ((p.dv + gds::kCols - 1) / gds::kCols) < (1LL << 32) / 256, "problem too large");   // (threads of a launch)
    VMS_CHECK(p.state && p.q && p.k && p.v && p.g && p.beta && p.out, "state, q, k, v, g, beta, out are required");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p.state_dtype == VMS_F32) gds::launch<float>(p, s);
    else if (p.state_dtype == VMS_F16) gds::launch<f16_t>(p, s);
    else gds::launch<bf16_t>(p, s);
    VMS_LAUNCH_CHECK();
    set_last_kernel("gated_delta_step");
    return VMS_OK;
}
extern "C" int vms_sizeof_gated_delta_step_params(void) { return (int)sizeof(vms_gated_delta_step_params); }
