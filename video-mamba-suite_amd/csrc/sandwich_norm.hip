// sandwich_norm.hip -- the norm after a block, its gate, the scaled residual add and the norm before the next block, one pass each way:
//   h = norm(x; w1, b1);  r' = residual_scale * r + gate * h;  y = norm(r'; w2, b2)
// Streaming kernels (forward: x, r in, y, r' out; backward: x, r, dy, dr' in, dx, dr out) with two dependent row reductions.  A row
// belongs to a team of 64, 256 or 1024 lanes (8 or 16 columns a lane, all of the row's values in registers from the load to the store);
// one wave per row as long as that fits (cols <= 1024), since its reductions are DPP sums without barriers.  Statistics are two-pass in fp32
// (mean first, then squares of differences).  y is the norm of the sum before it is rounded to the stream's type; the backward rebuilds that
// sum from x and r (the bytes of reading r' instead) and the four saved statistics of a row.
// Sums over rows (dw, db, dgate): in registers over the rows a team walks, one partial row per workgroup, a finish launch adds them in a fixed order.
//   P1 = sum dr * xhat1, P0 = sum dr of the rows that share a gate row:  dgate = w1 P1 + b1 P0, dw1 = sum gate P1, db1 = sum gate P0
#include "vms_common.h"

namespace vms {
namespace sn {

template <typename T>
__device__ __forceinline__ void ld8(const T* row, int c, int n, float (&o)[8]) {
    T v[8];
    if (c + 8 <= n) __builtin_memcpy(v, row + c, sizeof(v));
    else
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < n ? row[c + e] : static_cast<T>(0.f);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = static_cast<float>(v[e]);
}
template <typename T>
__device__ __forceinline__ void st8(T* row, int c, int n, const float (&o)[8]) {
    T v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = static_cast<T>(o[e]);
    if (c + 8 <= n) __builtin_memcpy(row + c, v, sizeof(v));
    else
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < n) row[c + e] = v[e];
}
__device__ __forceinline__ void ld8_any(const void* base, int64_t row, int c, int n, int dt, float (&o)[8]) {
    if (dt == VMS_F32) ld8<float>(static_cast<const float*>(base) + row, c, n, o);
    else if (dt == VMS_F16) ld8<f16_t>(static_cast<const f16_t*>(base) + row, c, n, o);
    else ld8<bf16_t>(static_cast<const bf16_t*>(base) + row, c, n, o);
}
__device__ __forceinline__ void st8_any(void* base, int64_t row, int c, int n, int dt, const float (&o)[8]) {
    if (dt == VMS_F32) st8<float>(static_cast<float*>(base) + row, c, n, o);
    else if (dt == VMS_F16) st8<f16_t>(static_cast<f16_t*>(base) + row, c, n, o);
    else st8<bf16_t>(static_cast<bf16_t*>(base) + row, c, n, o);
}

// sums over a team; red: 2 x 2 x 16 floats of LDS, used in turn so that one barrier per sum is enough
template <int TS>
struct Team {
    float* red;
    int turn = 0;
    __device__ __forceinline__ void sum2(float& a, float& b) {
        a = wave_sum(a);
        b = wave_sum(b);
        if constexpr (TS > 64) {
            float* const r = red + 32 * turn;
            turn ^= 1;
            const int w = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) { r[w] = a; r[16 + w] = b; }
            __syncthreads();
            a = 0.f; b = 0.f;
#pragma unroll
            for (int i = 0; i < TS / 64; ++i) { a += r[i]; b += r[16 + i]; }
        }
    }
    __device__ __forceinline__ float sum(float a) {
        float z = 0.f;
        if constexpr (TS > 64) sum2(a, z);
        else a = wave_sum(a);
        return a;
    }
};

template <typename TX, typename TR, bool RMS, int TS, int K>
__global__ __launch_bounds__(TS < 256 ? 256 : TS) void sandwich_fwd_kernel(const vms_sandwich_norm_params p) {
    constexpr int TEAMS = TS == 64 ? 4 : 1;
    __shared__ float red[64];
    Team<TS> team{red};
    const int lane = threadIdx.x % TS, N = p.cols;
    const float inv_n = 1.f / N;
    for (int64_t row = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TS; row < p.rows; row += (int64_t)gridDim.x * TEAMS) {
        const TX* const x = static_cast<const TX*>(p.x) + row * p.x_row_stride;
        float v[K][8], r[K][8];
#pragma unroll
        for (int k = 0; k < K; ++k) ld8<TX>(x, 8 * (lane + TS * k), N, v[k]);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (p.residual) ld8<TR>(static_cast<const TR*>(p.residual) + row * p.residual_row_stride, 8 * (lane + TS * k), N, r[k]);
            else
                for (int e = 0; e < 8; ++e) r[k][e] = 0.f;
        }
        auto norm = [&](float (&z)[K][8], float& mean, float& rstd) __attribute__((always_inline)) {
            mean = 0.f;
            if constexpr (!RMS) {
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) s += z[k][e];   // zeros behind the row's end
                mean = team.sum(s) * inv_n;
            }
            float q = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool in = 8 * (lane + TS * k) + e < N;
                    z[k][e] = in ? z[k][e] - mean : 0.f;
                    q = fmaf(z[k][e], z[k][e], q);
                }
            rstd = 1.f / sqrtf(team.sum(q) * inv_n + p.eps);
        };
        float m1, s1, m2, s2;
        norm(v, m1, s1);
        const int64_t gate_row = p.gate ? row / p.rows_per_gate * p.gate_row_stride : 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = 8 * (lane + TS * k);
            if (c < N) {
                float w[8], b[8], g[8];
                ld8<float>(p.post_weight, c, N, w);
                if (p.post_bias) ld8<float>(p.post_bias, c, N, b);
                if (p.gate) ld8_any(p.gate, gate_row, c, N, p.gate_dtype, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float h = v[k][e] * s1 * w[e];
                    if (p.post_bias) h += b[e];
                    if (p.gate) h *= g[e];
                    r[k][e] = c + e < N ? fmaf(p.residual_scale, r[k][e], h) : 0.f;
                }
                st8<TR>(static_cast<TR*>(p.residual_out) + row * p.residual_out_row_stride, c, N, r[k]);
            }
        }
        norm(r, m2, s2);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = 8 * (lane + TS * k);
            if (c < N) {
                float w[8], b[8];
                ld8<float>(p.pre_weight, c, N, w);
                if (p.pre_bias) ld8<float>(p.pre_bias, c, N, b);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    r[k][e] *= s2 * w[e];
                    if (p.pre_bias) r[k][e] += b[e];
                }
                st8<TX>(static_cast<TX*>(p.y) + row * p.y_row_stride, c, N, r[k]);
            }
        }
        if (p.stats && lane == 0) *reinterpret_cast<float4*>(p.stats + 4 * row) = make_float4(m1, s1, m2, s2);
    }
}

// Which rows a workgroup walks.  groups = gate rows that collect sums (1 without a gate, or with one of a row per token, whose gradient is
// written row by row).  Few groups: `parts` workgroups share each (whole = 0).  More groups than workgroups: a team walks whole groups (whole = 1).
struct Plan { int groups, parts, whole, partials; int64_t rpg; };
constexpr int kMostWgs = 1024;   // 4 per CU
static int team_size(int cols) { return cols <= 1024 ? 64 : cols <= 4096 ? 256 : 1024; }
static Plan plan_of(const vms_sandwich_norm_params& p) {
    Plan l{};
    l.rpg = p.gate && p.rows_per_gate > 1 ? p.rows_per_gate : p.rows;
    l.groups = (int)(p.rows / l.rpg);
    const int teams = team_size(p.cols) == 64 ? 4 : 1;
    l.whole = l.groups > kMostWgs / 2;
    if (l.whole) {
        const int want = (l.groups + teams - 1) / teams;
        l.parts = 1;
        l.partials = want < kMostWgs ? want : kMostWgs;
    } else {
        const int64_t most = (l.rpg + teams - 1) / teams;
        l.parts = kMostWgs / l.groups;
        if (l.parts > most) l.parts = (int)most;
        l.partials = l.groups * l.parts;
    }
    return l;
}

template <typename TX, typename TR, bool RMS, int TS, int K>
__global__ __launch_bounds__(TS < 256 ? 256 : TS) void sandwich_bwd_kernel(const vms_sandwich_norm_bwd_params q, const Plan plan) {
    constexpr int TEAMS = TS == 64 ? 4 : 1;
    __shared__ float red[64];
    __shared__ float sums[TEAMS > 1 ? (TEAMS - 1) * K * 8 * 64 : 1];
    const vms_sandwich_norm_params& p = q.f;
    Team<TS> team{red};
    const int lane = threadIdx.x % TS, tm = threadIdx.x / TS, N = p.cols;
    const float inv_n = 1.f / N;
    const bool row_gate = p.gate && p.rows_per_gate == 1, col_gate = p.gate && p.rows_per_gate > 1;
    float P1[K][8], P0[K][8], Q1[K][8], Q0[K][8];   // sums over this team's rows
    float A1[K][8], A0[K][8];                        // whole groups: the gate-weighted sums of P1, P0
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) { P1[k][e] = 0.f; P0[k][e] = 0.f; Q1[k][e] = 0.f; Q0[k][e] = 0.f; A1[k][e] = 0.f; A0[k][e] = 0.f; }

    auto one_row = [&](int64_t row) __attribute__((always_inline)) {
        const float4 st = *reinterpret_cast<const float4*>(p.stats + 4 * row);
        float xh[K][8], rh[K][8], t[K][8], dr[K][8];
        const int64_t gate_row = p.gate ? row / p.rows_per_gate * p.gate_row_stride : 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = 8 * (lane + TS * k);
            ld8<TX>(static_cast<const TX*>(p.x) + row * p.x_row_stride, c, N, xh[k]);
            if (p.residual) ld8<TR>(static_cast<const TR*>(p.residual) + row * p.residual_row_stride, c, N, rh[k]);
            else
                for (int e = 0; e < 8; ++e) rh[k][e] = 0.f;
            if (q.dy) ld8<TX>(static_cast<const TX*>(q.dy) + row * q.dy_row_stride, c, N, t[k]);
            else
                for (int e = 0; e < 8; ++e) t[k][e] = 0.f;
            if (q.dresidual_out) ld8<TR>(static_cast<const TR*>(q.dresidual_out) + row * q.dresidual_out_row_stride, c, N, dr[k]);
            else
                for (int e = 0; e < 8; ++e) dr[k][e] = 0.f;
        }
        float g[K][8], w1[K][8];
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = 8 * (lane + TS * k);
            float b[8], w2[8];
            ld8<float>(p.post_weight, c, N, w1[k]);
            ld8<float>(p.pre_weight, c, N, w2);
            if (p.post_bias) ld8<float>(p.post_bias, c, N, b);
            if (p.gate) ld8_any(p.gate, gate_row, c, N, p.gate_dtype, g[k]);
            float dg[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = c + e < N;
                xh[k][e] = in ? (xh[k][e] - st.x) * st.y : 0.f;
                float h = xh[k][e] * w1[k][e];
                if (p.post_bias) h += b[e];
                dg[e] = h;
                if (p.gate) h *= g[k][e];
                rh[k][e] = in ? (fmaf(p.residual_scale, rh[k][e], h) - st.z) * st.w : 0.f;
                Q1[k][e] = fmaf(t[k][e], rh[k][e], Q1[k][e]);
                Q0[k][e] += t[k][e];
                t[k][e] *= w2[e];
                c1 = fmaf(t[k][e], rh[k][e], c1);
                c2 += t[k][e];
            }
        }
        team.sum2(c1, c2);
        c1 *= inv_n;
        c2 = RMS ? 0.f : c2 * inv_n;
        float d1 = 0.f, d2 = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = 8 * (lane + TS * k);
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = c + e < N ? fmaf(t[k][e] - fmaf(rh[k][e], c1, c2), st.w, dr[k][e]) : 0.f;
                dr[k][e] = d;
                o[e] = p.residual_scale * d;
            }
            if (q.dresidual && c < N) st8<TR>(static_cast<TR*>(q.dresidual) + row * q.dresidual_row_stride, c, N, o);
            if (row_gate && c < N) {
                float b[8];
                if (p.post_bias) ld8<float>(p.post_bias, c, N, b);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = dr[k][e] * (p.post_bias ? fmaf(xh[k][e], w1[k][e], b[e]) : xh[k][e] * w1[k][e]);
                if (q.dgate) st8_any(q.dgate, row * (int64_t)N, c, N, p.gate_dtype, o);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float d = dr[k][e];
                if (!col_gate && p.gate) d *= g[k][e];   // a row's own gate enters the sums here, a shared one afterwards
                P1[k][e] = fmaf(d, xh[k][e], P1[k][e]);
                P0[k][e] += d;
                if (col_gate) d *= g[k][e];
                d *= w1[k][e];
                t[k][e] = d;
                d1 = fmaf(d, xh[k][e], d1);
                d2 += d;
            }
        }
        team.sum2(d1, d2);
        d1 *= inv_n;
        d2 = RMS ? 0.f : d2 * inv_n;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = 8 * (lane + TS * k);
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = (t[k][e] - fmaf(xh[k][e], d1, d2)) * st.y;
            if (c < N) st8<TX>(static_cast<TX*>(q.dx) + row * q.dx_row_stride, c, N, o);
        }
    };

    if (!plan.whole) {
        const int64_t first = (int64_t)(blockIdx.x / plan.parts) * plan.rpg;
        for (int64_t i = (int64_t)(blockIdx.x % plan.parts) * TEAMS + tm; i < plan.rpg; i += (int64_t)plan.parts * TEAMS) one_row(first + i);
    } else {
        for (int64_t gr = (int64_t)blockIdx.x * TEAMS + tm; gr < plan.groups; gr += (int64_t)gridDim.x * TEAMS) {
            for (int64_t i = 0; i < plan.rpg; ++i) one_row(gr * plan.rpg + i);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = 8 * (lane + TS * k);
                if (c < N) {
                    float w[8], b[8], g[8], o[8];
                    ld8<float>(p.post_weight, c, N, w);
                    if (p.post_bias) ld8<float>(p.post_bias, c, N, b);
                    ld8_any(p.gate, gr * p.gate_row_stride, c, N, p.gate_dtype, g);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        o[e] = w[e] * P1[k][e] + (p.post_bias ? b[e] * P0[k][e] : 0.f);
                        A1[k][e] = fmaf(g[e], P1[k][e], A1[k][e]);
                        A0[k][e] = fmaf(g[e], P0[k][e], A0[k][e]);
                        P1[k][e] = 0.f;
                        P0[k][e] = 0.f;
                    }
                    if (q.dgate) st8_any(q.dgate, gr * (int64_t)N, c, N, p.gate_dtype, o);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) { P1[k][e] = A1[k][e]; P0[k][e] = A0[k][e]; }
    }
    float* const out = static_cast<float*>(q.workspace) + (int64_t)blockIdx.x * 4 * N;
    auto emit = [&](float (&a)[K][8], int which) __attribute__((always_inline)) {
        if constexpr (TEAMS > 1) {
            __syncthreads();
            if (tm > 0)
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) sums[((tm - 1) * K * 8 + k * 8 + e) * 64 + lane] = a[k][e];
            __syncthreads();
        }
        if (tm == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = 8 * (lane + TS * k);
                if constexpr (TEAMS > 1)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
#pragma unroll
                        for (int t2 = 0; t2 < TEAMS - 1; ++t2) a[k][e] += sums[(t2 * K * 8 + k * 8 + e) * 64 + lane];
                if (c < N) st8<float>(out + (int64_t)which * N, c, N, a[k]);
            }
    };
    emit(P1, 0);
    emit(P0, 1);
    emit(Q1, 2);
    emit(Q0, 3);
}

// ---- the partial rows' sums.  A workgroup owns 16 columns, 64 row lanes x 4 column groups.  blockIdx.y < gate_rows: dgate of that gate row
// from its `parts` partial rows; the last y: dw1, db1 (with the gate of each partial row's group where `weigh`), dw2, db2
__global__ __launch_bounds__(256) void sandwich_finish_kernel(const vms_sandwich_norm_bwd_params q, const Plan plan, const int gate_rows, const int weigh) {
    __shared__ float red[4][64][17];
    const vms_sandwich_norm_params& p = q.f;
    const int N = p.cols, rl = threadIdx.x >> 2, cg = threadIdx.x & 3, c0 = blockIdx.x * 16 + 4 * cg;
    const bool weights = (int)blockIdx.y == gate_rows;
    const float* const src = static_cast<const float*>(q.workspace);
    const int r0 = weights ? 0 : blockIdx.y * plan.parts, r1 = weights ? plan.partials : r0 + plan.parts, arrays = weights ? 4 : 2;
    float a[4][4] = {};
    for (int r = r0 + rl; r < r1; r += 64)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = c0 + e;
            if (c < N) {
                const float* const row = src + (int64_t)r * 4 * N + c;
                float g = 1.f;
                if (weights && weigh) {
                    const int64_t at = (int64_t)(r / plan.parts) * p.gate_row_stride + c;
                    g = p.gate_dtype == VMS_F32 ? static_cast<const float*>(p.gate)[at]
                        : p.gate_dtype == VMS_F16 ? static_cast<float>(static_cast<const f16_t*>(p.gate)[at]) : static_cast<float>(static_cast<const bf16_t*>(p.gate)[at]);
                }
                a[0][e] = fmaf(g, row[0], a[0][e]);
                a[1][e] = fmaf(g, row[N], a[1][e]);
                if (arrays == 4) {
                    a[2][e] += row[2 * (int64_t)N];
                    a[3][e] += row[3 * (int64_t)N];
                }
            }
        }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[i][rl][4 * cg + e] = a[i][e];
    __syncthreads();
    if (threadIdx.x < 64) {
        const int i = threadIdx.x >> 4, cc = threadIdx.x & 15, c = blockIdx.x * 16 + cc;
        float t = 0.f;
#pragma unroll 8
        for (int r = 0; r < 64; ++r) t += red[i][r][cc];
        if (weights) {
            float* const dst = i == 0 ? q.dpost_weight : i == 1 ? q.dpost_bias : i == 2 ? q.dpre_weight : q.dpre_bias;
            if (dst && c < N) dst[c] = t;
        } else {
            const float p0 = __shfl(t, 16 + cc);   // i == 0 holds the sum of P1, i == 1 that of P0
            if (i == 0 && c < N) {
                const float d = p.post_weight[c] * t + (p.post_bias ? p.post_bias[c] * p0 : 0.f);
                const int64_t at = (int64_t)blockIdx.y * N + c;
                if (p.gate_dtype == VMS_F32) static_cast<float*>(q.dgate)[at] = d;
                else if (p.gate_dtype == VMS_F16) static_cast<f16_t*>(q.dgate)[at] = static_cast<f16_t>(d);
                else static_cast<bf16_t*>(q.dgate)[at] = static_cast<bf16_t>(d);
            }
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------
static int validate(const vms_sandwich_norm_params& p) {
    auto dt_ok = [](int d) { return d == VMS_F32 || d == VMS_F16 || d == VMS_BF16; };
    VMS_CHECK(dt_ok(p.x_dtype) && dt_ok(p.res_dtype), "dtypes must be fp32/fp16/bf16");
    VMS_CHECK(p.res_dtype == p.x_dtype || p.res_dtype == VMS_F32, "the residual stream must be fp32 or of the type of x");
    VMS_CHECK(p.rows > 0 && p.cols > 0, "empty problem");
    VMS_CHECK(p.cols <= 8192, "rows of up to 8192");
    VMS_CHECK(p.x && p.post_weight && p.pre_weight, "x, post_weight, pre_weight are required");
    VMS_CHECK(aligned16(p.stats), "stats must be 16-byte aligned");
    if (p.gate) {
        VMS_CHECK(dt_ok(p.gate_dtype), "gate dtype must be fp32/fp16/bf16");
        VMS_CHECK(p.rows_per_gate >= 1 && p.rows % p.rows_per_gate == 0, "rows must be a multiple of rows_per_gate");
    }
    return VMS_OK;
}

template <typename TX, typename TR, bool RMS>
static int fwd_launch(const vms_sandwich_norm_params& p, hipStream_t s) {
    const int ts = team_size(p.cols);
    const int64_t want = ts == 64 ? (p.rows + 3) / 4 : p.rows;
    const dim3 grid((unsigned)(want < 2048 ? want : 2048)), block(ts < 256 ? 256 : ts);
    if (p.cols <= 512) hipLaunchKernelGGL((sandwich_fwd_kernel<TX, TR, RMS, 64, 1>), grid, block, 0, s, p);
    else if (ts == 64) hipLaunchKernelGGL((sandwich_fwd_kernel<TX, TR, RMS, 64, 2>), grid, block, 0, s, p);
    else if (p.cols <= 2048) hipLaunchKernelGGL((sandwich_fwd_kernel<TX, TR, RMS, 256, 1>), grid, block, 0, s, p);
    else if (ts == 256) hipLaunchKernelGGL((sandwich_fwd_kernel<TX, TR, RMS, 256, 2>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((sandwich_fwd_kernel<TX, TR, RMS, 1024, 1>), grid, block, 0, s, p);
    VMS_LAUNCH_CHECK();
    return VMS_OK;
}
template <typename TX, typename TR, bool RMS>
static int bwd_launch(const vms_sandwich_norm_bwd_params& q, hipStream_t s) {
    const vms_sandwich_norm_params& p = q.f;
    const Plan plan = plan_of(p);
    const int ts = team_size(p.cols);
    const dim3 grid(plan.partials), block(ts < 256 ? 256 : ts);
    if (p.cols <= 512) hipLaunchKernelGGL((sandwich_bwd_kernel<TX, TR, RMS, 64, 1>), grid, block, 0, s, q, plan);
    else if (ts == 64) hipLaunchKernelGGL((sandwich_bwd_kernel<TX, TR, RMS, 64, 2>), grid, block, 0, s, q, plan);
    else if (p.cols <= 2048) hipLaunchKernelGGL((sandwich_bwd_kernel<TX, TR, RMS, 256, 1>), grid, block, 0, s, q, plan);
    else if (ts == 256) hipLaunchKernelGGL((sandwich_bwd_kernel<TX, TR, RMS, 256, 2>), grid, block, 0, s, q, plan);
    else hipLaunchKernelGGL((sandwich_bwd_kernel<TX, TR, RMS, 1024, 1>), grid, block, 0, s, q, plan);
    VMS_LAUNCH_CHECK();
    const bool col_gate = p.gate && p.rows_per_gate > 1;
    const int gate_rows = col_gate && !plan.whole && q.dgate ? plan.groups : 0;
    hipLaunchKernelGGL(sandwich_finish_kernel, dim3((p.cols + 15) / 16, gate_rows + 1), dim3(256), 0, s, q, plan, gate_rows, col_gate && !plan.whole ? 1 : 0);
    VMS_LAUNCH_CHECK();
    return VMS_OK;
}

#define VMS_SN_DISPATCH(FN, P_, ARG, s)                                                                                                  \
    do {                                                                                                                                 \
        const bool f32_ = (P_).res_dtype == VMS_F32, rms_ = (P_).is_rms != 0;                                                            \
        switch ((P_).x_dtype) {                                                                                                          \
            case VMS_F32: rc = rms_ ? FN<float, float, true>(ARG, s) : FN<float, float, false>(ARG, s); break;                           \
            case VMS_F16:                                                                                                                \
                rc = f32_ ? (rms_ ? FN<f16_t, float, true>(ARG, s) : FN<f16_t, float, false>(ARG, s))                                    \
                          : (rms_ ? FN<f16_t, f16_t, true>(ARG, s) : FN<f16_t, f16_t, false>(ARG, s));                                   \
                break;                                                                                                                   \
            default:                                                                                                                     \
                rc = f32_ ? (rms_ ? FN<bf16_t, float, true>(ARG, s) : FN<bf16_t, float, false>(ARG, s))                                  \
                          : (rms_ ? FN<bf16_t, bf16_t, true>(ARG, s) : FN<bf16_t, bf16_t, false>(ARG, s));                               \
        }                                                                                                                                \
    } while (0)

}  // namespace sn
}  // namespace vms

using namespace vms;

extern "C" int vms_sandwich_norm_fwd(const vms_sandwich_norm_params* pp, void* stream) {
    VMS_CHECK(pp != nullptr, "null params");
    const vms_sandwich_norm_params& p = *pp;
    if (int rc = sn::validate(p)) return rc;
    VMS_CHECK(p.y && p.residual_out, "y and residual_out are required");
    int rc = VMS_OK;
    VMS_SN_DISPATCH(sn::fwd_launch, p, p, static_cast<hipStream_t>(stream));
    if (rc == VMS_OK) set_last_kernel("sandwich_norm_fwd");
    return rc;
}
extern "C" int64_t vms_sandwich_norm_bwd_workspace_bytes(const vms_sandwich_norm_params* pp) {
    if (!pp || pp->rows <= 0 || pp->cols <= 0 || pp->cols > 8192 || (pp->gate && pp->rows_per_gate < 1)) return 0;
    return (int64_t)sn::plan_of(*pp).partials * 4 * pp->cols * 4;
}
extern "C" int vms_sandwich_norm_bwd(const vms_sandwich_norm_bwd_params* qq, void* stream) {
    VMS_CHECK(qq != nullptr, "null params");
    const vms_sandwich_norm_bwd_params& q = *qq;
    if (int rc = sn::validate(q.f)) return rc;
    VMS_CHECK(q.f.stats && q.dx && q.dpost_weight && q.dpre_weight, "stats, dx, dpost_weight, dpre_weight are required");
    VMS_CHECK(!q.f.gate || q.dgate, "dgate comes with gate");
    VMS_CHECK(q.workspace && q.workspace_bytes >= vms_sandwich_norm_bwd_workspace_bytes(&q.f), "workspace is too small (vms_sandwich_norm_bwd_workspace_bytes)");
    int rc = VMS_OK;
    VMS_SN_DISPATCH(sn::bwd_launch, q.f, q, static_cast<hipStream_t>(stream));
    if (rc == VMS_OK) set_last_kernel("sandwich_norm_bwd");
    return rc;
}
extern "C" int vms_sizeof_sandwich_norm_params(void) { return (int)sizeof(vms_sandwich_norm_params); }
extern "C" int vms_sizeof_sandwich_norm_bwd_params(void) { return (int)sizeof(vms_sandwich_norm_bwd_params); }
