// sandwich_norm.hip -- the norm after a block, its gate, the scaled residual add and the norm before the next block, one pass each way:
//   h = norm(x; w1, b1);  r' = residual_scale * r + gate * h;  y = norm(r'; w2, b2)
// Streaming kernels (forward: x, r in, y, r' out; backward: x, r, dy, dr' in, dx, dr out) with two dependent row reductions.  A row
// belongs to a team of lanes (forward: 8 or 16 columns a lane, one wave up to 1024 columns, whose reductions are DPP sums without barriers; backward: 8 a
// lane, its sums over rows want the registers), all of its values in registers from the load to the store.  Statistics are two-pass in fp32
// (mean first, then squares of differences).  y is the norm of the sum before it is rounded to the stream's type; the backward rebuilds that
// sum from x and r (the bytes of reading r' instead) and the four saved statistics of a row.
// Sums over rows (dw, db, dgate): in registers over the rows a team walks, one partial row per workgroup, a finish launch adds them in a fixed order.
//   P1 = sum dr * xhat1, P0 = sum dr of the rows that share a gate row:  dgate = w1 P1 + b1 P0, dw1 = sum gate P1, db1 = sum gate P0
#include "vms_common.h"

namespace vms {
namespace sn {

// 16 bytes at any alignment
typedef unsigned __attribute__((ext_vector_type(4), aligned(2))) u4_any;

// 8 columns c .. c+7 of a row of n, any alignment; zeros outside.  WHOLE: n % 8 == 0.  No branch around a load (its registers would be written by the other side
// too, and the wave would wait for each load before the next), and zeros are put in word by word (element by element the compiler takes the load apart).
template <bool WHOLE, typename T>
__device__ __forceinline__ void ld8(const T* row, int c, int n, float (&o)[8]) {
    constexpr int V = sizeof(T) / 2;   // 16-byte vectors
    if constexpr (WHOLE) {
        const u4_any* const at = reinterpret_cast<const u4_any*>(row + (c < n ? c : 0));
        unsigned w[4 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const u4_any x = at[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[4 * i + e] = x[e];
        }
#pragma unroll
        for (int i = 0; i < 4 * V; ++i) w[i] = c < n ? w[i] : 0u;
        T v[8];
        __builtin_memcpy(v, w, sizeof(v));
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = static_cast<float>(v[e]);
    } else {
        T v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = row[c + e < n ? c + e : 0];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = c + e < n ? static_cast<float>(v[e]) : 0.f;
    }
}
template <bool WHOLE, typename T>   // c < n
__device__ __forceinline__ void st8(T* row, int c, int n, const float (&o)[8]) {
    T v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = static_cast<T>(o[e]);
    if constexpr (WHOLE) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            vec_t<unsigned, 4> x;
            __builtin_memcpy(&x, reinterpret_cast<const char*>(v) + 16 * i, 16);
            reinterpret_cast<u4_any*>(row + c)[i] = x;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < n) row[c + e] = v[e];
    }
}
template <bool WHOLE>
__device__ __forceinline__ void ld8_any(const void* base, int64_t row, int c, int n, int dt, float (&o)[8]) {
    if (dt == VMS_F32) ld8<WHOLE, float>(static_cast<const float*>(base) + row, c, n, o);
    else if (dt == VMS_F16) ld8<WHOLE, f16_t>(static_cast<const f16_t*>(base) + row, c, n, o);
    else ld8<WHOLE, bf16_t>(static_cast<const bf16_t*>(base) + row, c, n, o);
}
template <bool WHOLE>
__device__ __forceinline__ void st8_any(void* base, int64_t row, int c, int n, int dt, const float (&o)[8]) {
    if (dt == VMS_F32) st8<WHOLE, float>(static_cast<float*>(base) + row, c, n, o);
    else if (dt == VMS_F16) st8<WHOLE, f16_t>(static_cast<f16_t*>(base) + row, c, n, o);
    else st8<WHOLE, bf16_t>(static_cast<bf16_t*>(base) + row, c, n, o);
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

template <typename TX, typename TR, int TS, int K, bool WHOLE>
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
        for (int k = 0; k < K; ++k) ld8<WHOLE, TX>(x, 8 * (lane + TS * k), N, v[k]);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (p.residual) ld8<WHOLE, TR>(static_cast<const TR*>(p.residual) + row * p.residual_row_stride, 8 * (lane + TS * k), N, r[k]);
            else
                for (int e = 0; e < 8; ++e) r[k][e] = 0.f;
        }
        auto norm = [&](float (&z)[K][8], float& mean, float& rstd) __attribute__((always_inline)) {
            mean = 0.f;
            if (!p.is_rms) {
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
                ld8<WHOLE, float>(p.post_weight, c, N, w);
                if (p.post_bias) ld8<WHOLE, float>(p.post_bias, c, N, b);
                if (p.gate) ld8_any<WHOLE>(p.gate, gate_row, c, N, p.gate_dtype, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float h = v[k][e] * s1 * w[e];
                    if (p.post_bias) h += b[e];
                    if (p.gate) h *= g[e];
                    r[k][e] = c + e < N ? fmaf(p.residual_scale, r[k][e], h) : 0.f;
                }
                st8<WHOLE, TR>(static_cast<TR*>(p.residual_out) + row * p.residual_out_row_stride, c, N, r[k]);
            }
        }
        norm(r, m2, s2);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = 8 * (lane + TS * k);
            if (c < N) {
                float w[8], b[8];
                ld8<WHOLE, float>(p.pre_weight, c, N, w);
                if (p.pre_bias) ld8<WHOLE, float>(p.pre_bias, c, N, b);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    r[k][e] *= s2 * w[e];
                    if (p.pre_bias) r[k][e] += b[e];
                }
                st8<WHOLE, TX>(static_cast<TX*>(p.y) + row * p.y_row_stride, c, N, r[k]);
            }
        }
        if (p.stats && lane == 0) *reinterpret_cast<float4*>(p.stats + 4 * row) = make_float4(m1, s1, m2, s2);
    }
}

// Which rows a workgroup walks.  groups = gate rows that collect sums (1 without a gate, or with one of a row per token, whose gradient is
// written row by row).  `parts` workgroups share each (whole = 0), or a team walks whole groups (whole = 1).  A team's rows follow one another (about 2 us each), which
// many teams hide; shared groups leave a partial row each, which the finish reads.  Both sides, backward of one call, us (shared / whole; bf16, fp32 stream, biases):
//   groups          64 columns, 16 rows   64 columns, 196   384 columns, 4   384 columns, 64   768 columns, 16   1536 columns, 64   3000 columns, 4
//   128                  18 / 31              59 / 383          12 / 14           43 / 142          49 / 43           79 / 184           45 / 25
//   512                  35 / 32             142 / 403          21 / 16           79 / 144          63 / 53          327 / 273          129 / 52
//   1024                 42 / 34             257 / 404          37 / 20          168 / 208          95 / 78          640 / 594          237 / 117
//   2048                 81 / 51             519 / 568          67 / 25          279 / 260         232 / 162              -             478 / 209
// The rule sets a team's chain against what all groups cost together, rows and partial rows.  Over 6 widths, 2 to 784 rows and 128 to 16384 groups it is within a quarter
// of the better side, but at 128 groups of 768 columns and 4 rows, and of 3000 columns and 16 rows (a third).
struct Plan { int groups, parts, whole, partials; int64_t rpg; };
constexpr int kMostWgs = 1024;   // 4 per CU
// lanes of a row in the backward: 8 columns each
static int team_of(int cols) { return cols <= 512 ? 64 : cols <= 1024 ? 128 : cols <= 2048 ? 256 : cols <= 4096 ? 512 : 1024; }
static Plan plan_of(const vms_sandwich_norm_params& p) {
    Plan l{};
    l.rpg = p.gate && p.rows_per_gate > 1 ? p.rows_per_gate : p.rows;
    l.groups = (int)(p.rows / l.rpg);
    const int ts = team_of(p.cols), teams = ts == 64 ? 4 : 1, most_wgs = ts == 128 ? 3 * kMostWgs / 2 : kMostWgs;   // (as many as are resident)
    l.whole = l.groups > 1 && l.groups * (l.rpg * (270 + p.cols) + 16000 + 14 * p.cols) > 1300000 * l.rpg;   // (shared: fewer than 4800)
    if (l.whole) {
        const int want = (l.groups + teams - 1) / teams;
        l.parts = 1;
        l.partials = want < most_wgs ? want : most_wgs;
    } else {
        const int64_t most = (l.rpg + teams - 1) / teams;
        l.parts = l.groups < most_wgs ? most_wgs / l.groups : 1;
        if (l.parts > most) l.parts = (int)most;
        l.partials = l.groups * l.parts;
    }
    return l;
}

// GROUPS: whole groups per team (Plan::whole)
template <typename TX, typename TR, int TS, bool WHOLE, bool GROUPS>
__global__ __launch_bounds__(TS < 128 ? 256 : TS, TS == 1024 ? 4 : 3) void sandwich_bwd_kernel(const vms_sandwich_norm_bwd_params q, const Plan plan) {
    constexpr int TEAMS = TS == 64 ? 4 : 1;
    __shared__ float red[64];
    __shared__ float sums[TEAMS > 1 ? (TEAMS - 1) * 8 * 64 : 1];
    const vms_sandwich_norm_params& p = q.f;
    Team<TS> team{red};
    const int lane = threadIdx.x % TS, tm = threadIdx.x / TS, N = p.cols, c = 8 * lane;
    const float inv_n = 1.f / N, center = p.is_rms ? 0.f : inv_n;
    const bool row_gate = p.gate && p.rows_per_gate == 1, col_gate = p.gate && p.rows_per_gate > 1;
    float P1[8] = {}, P0[8] = {}, Q1[8] = {}, Q0[8] = {};   // sums over this team's rows
    float A1[GROUPS ? 8 : 1] = {}, A0[GROUPS ? 8 : 1] = {};   // whole groups: the gate-weighted sums of P1, P0

    auto one_row = [&](int64_t row) __attribute__((always_inline)) {
        const float4 st = *reinterpret_cast<const float4*>(p.stats + 4 * row);
        float xh[8], rh[8] = {}, t[8] = {}, dr[8] = {}, g[8], w1[8], b[8] = {};
        const int64_t gate_row = p.gate ? row / p.rows_per_gate * p.gate_row_stride : 0;
        ld8<WHOLE, TX>(static_cast<const TX*>(p.x) + row * p.x_row_stride, c, N, xh);
        if (p.residual) ld8<WHOLE, TR>(static_cast<const TR*>(p.residual) + row * p.residual_row_stride, c, N, rh);
        if (q.dy) ld8<WHOLE, TX>(static_cast<const TX*>(q.dy) + row * q.dy_row_stride, c, N, t);
        if (q.dresidual_out) ld8<WHOLE, TR>(static_cast<const TR*>(q.dresidual_out) + row * q.dresidual_out_row_stride, c, N, dr);
        ld8<WHOLE, float>(p.post_weight, c, N, w1);
        if (p.post_bias) ld8<WHOLE, float>(p.post_bias, c, N, b);
        if (p.gate) ld8_any<WHOLE>(p.gate, gate_row, c, N, p.gate_dtype, g);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = 1.f;
        float w2[8];
        ld8<WHOLE, float>(p.pre_weight, c, N, w2);
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = c + e < N;
            xh[e] = in ? (xh[e] - st.x) * st.y : 0.f;
            const float h = fmaf(xh[e], w1[e], b[e]) * g[e];
            rh[e] = in ? (fmaf(p.residual_scale, rh[e], h) - st.z) * st.w : 0.f;
            Q1[e] = fmaf(t[e], rh[e], Q1[e]);
            Q0[e] += t[e];
            t[e] *= w2[e];
            c1 = fmaf(t[e], rh[e], c1);
            c2 += t[e];
        }
        team.sum2(c1, c2);
        c1 *= inv_n;
        c2 *= center;
        float d1 = 0.f, d2 = 0.f, o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dr[e] = c + e < N ? fmaf(t[e] - fmaf(rh[e], c1, c2), st.w, dr[e]) : 0.f;
            o[e] = p.residual_scale * dr[e];
        }
        if (q.dresidual && c < N) st8<WHOLE, TR>(static_cast<TR*>(q.dresidual) + row * q.dresidual_row_stride, c, N, o);
        if (row_gate && c < N) {
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = dr[e] * fmaf(xh[e], w1[e], b[e]);
            st8_any<WHOLE>(q.dgate, row * (int64_t)N, c, N, p.gate_dtype, o);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float gated = dr[e] * g[e];
            const float d = col_gate ? dr[e] : gated;   // a row's own gate enters the sums here, a shared one afterwards
            P1[e] = fmaf(d, xh[e], P1[e]);
            P0[e] += d;
            t[e] = gated * w1[e];
            d1 = fmaf(t[e], xh[e], d1);
            d2 += t[e];
        }
        team.sum2(d1, d2);
        d1 *= inv_n;
        d2 *= center;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (t[e] - fmaf(xh[e], d1, d2)) * st.y;
        if (c < N) st8<WHOLE, TX>(static_cast<TX*>(q.dx) + row * q.dx_row_stride, c, N, o);
    };

    if constexpr (!GROUPS) {
        const int64_t first = (int64_t)(blockIdx.x / plan.parts) * plan.rpg;
        for (int64_t i = (int64_t)(blockIdx.x % plan.parts) * TEAMS + tm; i < plan.rpg; i += (int64_t)plan.parts * TEAMS) one_row(first + i);
    } else {
        for (int64_t gr = (int64_t)blockIdx.x * TEAMS + tm; gr < plan.groups; gr += (int64_t)gridDim.x * TEAMS) {
            for (int64_t i = 0; i < plan.rpg; ++i) one_row(gr * plan.rpg + i);
            float w[8], b[8] = {}, g[8], o[8];
            ld8<WHOLE, float>(p.post_weight, c, N, w);
            if (p.post_bias) ld8<WHOLE, float>(p.post_bias, c, N, b);
            ld8_any<WHOLE>(p.gate, gr * p.gate_row_stride, c, N, p.gate_dtype, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                o[e] = fmaf(w[e], P1[e], b[e] * P0[e]);
                A1[e] = fmaf(g[e], P1[e], A1[e]);
                A0[e] = fmaf(g[e], P0[e], A0[e]);
                P1[e] = 0.f;
                P0[e] = 0.f;
            }
            if (c < N) st8_any<WHOLE>(q.dgate, gr * (int64_t)N, c, N, p.gate_dtype, o);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) { P1[e] = A1[e]; P0[e] = A0[e]; }
    }
    float* const out = static_cast<float*>(q.workspace) + (int64_t)blockIdx.x * 4 * N;
    auto emit = [&](float (&a)[8], int which) __attribute__((always_inline)) {
        if constexpr (TEAMS > 1) {
            __syncthreads();
            if (tm > 0)
#pragma unroll
                for (int e = 0; e < 8; ++e) sums[((tm - 1) * 8 + e) * 64 + lane] = a[e];
            __syncthreads();
            if (tm == 0)
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int t2 = 0; t2 < TEAMS - 1; ++t2) a[e] += sums[(t2 * 8 + e) * 64 + lane];
        }
        if (tm == 0 && c < N) st8<WHOLE, float>(out + (int64_t)which * N, c, N, a);
    };
    emit(P1, 0);
    emit(P0, 1);
    emit(Q1, 2);
    emit(Q0, 3);
}

// ---- the partial rows' sums.  A workgroup owns 64 columns (16 groups of 4) of one of the four arrays, 64 row lanes (with 16, one load at a time: 47 us
// for 1536 rows of 1024); blockIdx.y < 4: dw1, db1 (with the
// gate of each partial row's group where `weigh`), dw2, db2;  blockIdx.y >= 4: dgate of gate row y - 4 from its `parts` partial rows of P1 and P0
__global__ __launch_bounds__(1024) void sandwich_finish_kernel(const vms_sandwich_norm_bwd_params q, const Plan plan, const int weigh) {
    __shared__ float red[2][64][65];
    const vms_sandwich_norm_params& p = q.f;
    const int N = p.cols, rl = threadIdx.x >> 4, cg = threadIdx.x & 15, c0 = blockIdx.x * 64 + 4 * cg;
    const float* const src = static_cast<const float*>(q.workspace);
    const int z = blockIdx.y;
    const bool gate = z >= 4;
    const int r0 = gate ? (z - 4) * plan.parts : 0, r1 = gate ? r0 + plan.parts : plan.partials;
    const int which = gate ? 0 : z;
    float a[4] = {}, a2[4] = {};
    const bool vec = N % 4 == 0;
    auto ld4 = [&](const float* row, float (&v)[4]) __attribute__((always_inline)) {   // columns c0 .. c0 + 3
        if (vec) {
            const float4 x = *reinterpret_cast<const float4*>(row + (c0 < N ? c0 : 0));
            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = row[c0 + e < N ? c0 + e : 0];
        }
    };
    auto gate_at = [&](int64_t at) __attribute__((always_inline)) {
        return p.gate_dtype == VMS_F32 ? static_cast<const float*>(p.gate)[at]
               : p.gate_dtype == VMS_F16 ? static_cast<float>(static_cast<const f16_t*>(p.gate)[at]) : static_cast<float>(static_cast<const bf16_t*>(p.gate)[at]);
    };
    if (gate) {
#pragma unroll 4
        for (int r = r0 + rl; r < r1; r += 64) {
            float v[4], v2[4];
            ld4(src + (int64_t)r * 4 * N, v);
            ld4(src + (int64_t)r * 4 * N + N, v2);
#pragma unroll
            for (int e = 0; e < 4; ++e) { a[e] += v[e]; a2[e] += v2[e]; }
        }
    } else if (weigh && which < 2 && plan.groups > 1) {
#pragma unroll 4
        for (int r = r0 + rl; r < r1; r += 64) {
            float v[4];
            ld4(src + ((int64_t)r * 4 + which) * N, v);
            const int64_t at = (int64_t)(r / plan.parts) * p.gate_row_stride;
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = fmaf(gate_at(at + (c0 + e < N ? c0 + e : 0)), v[e], a[e]);
        }
    } else {
#pragma unroll 8
        for (int r = r0 + rl; r < r1; r += 64) {
            float v[4];
            ld4(src + ((int64_t)r * 4 + which) * N, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] += v[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) { red[0][rl][4 * cg + e] = a[e]; red[1][rl][4 * cg + e] = a2[e]; }
    __syncthreads();
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x < 64 && c < N) {
        float t = 0.f, t2 = 0.f;
#pragma unroll
        for (int r = 0; r < 64; ++r) { t += red[0][r][threadIdx.x]; t2 += red[1][r][threadIdx.x]; }
        if (!gate) {
            float* const dst = z == 0 ? q.dpost_weight : z == 1 ? q.dpost_bias : z == 2 ? q.dpre_weight : q.dpre_bias;
            if (dst) dst[c] = weigh && z < 2 && plan.groups == 1 ? t * gate_at(c) : t;   // (one gate row: a factor of the sum)
        } else {
            const float d = p.post_weight[c] * t + (p.post_bias ? p.post_bias[c] * t2 : 0.f);
            const int64_t at = (int64_t)(z - 4) * N + c;
            if (p.gate_dtype == VMS_F32) static_cast<float*>(q.dgate)[at] = d;
            else if (p.gate_dtype == VMS_F16) static_cast<f16_t*>(q.dgate)[at] = static_cast<f16_t>(d);
            else static_cast<bf16_t*>(q.dgate)[at] = static_cast<bf16_t>(d);
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

template <typename TX, typename TR, bool WHOLE>
static int fwd_launch(const vms_sandwich_norm_params& p, hipStream_t s) {
    const int ts = p.cols <= 1024 ? 64 : p.cols <= 4096 ? 256 : 1024;
    const int64_t want = ts == 64 ? (p.rows + 3) / 4 : p.rows;
    const dim3 grid((unsigned)(want < 2048 ? want : 2048)), block(ts < 256 ? 256 : ts);
    if (p.cols <= 512) hipLaunchKernelGGL((sandwich_fwd_kernel<TX, TR, 64, 1, WHOLE>), grid, block, 0, s, p);
    else if (ts == 64) hipLaunchKernelGGL((sandwich_fwd_kernel<TX, TR, 64, 2, WHOLE>), grid, block, 0, s, p);
    else if (p.cols <= 2048) hipLaunchKernelGGL((sandwich_fwd_kernel<TX, TR, 256, 1, WHOLE>), grid, block, 0, s, p);
    else if (ts == 256) hipLaunchKernelGGL((sandwich_fwd_kernel<TX, TR, 256, 2, WHOLE>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((sandwich_fwd_kernel<TX, TR, 1024, 1, WHOLE>), grid, block, 0, s, p);
    VMS_LAUNCH_CHECK();
    return VMS_OK;
}
template <typename TX, typename TR, bool WHOLE, bool GROUPS>
static void bwd_team(const vms_sandwich_norm_bwd_params& q, const Plan& plan, hipStream_t s) {
    const int ts = team_of(q.f.cols);
    const dim3 grid(plan.partials), block(ts == 64 ? 256 : ts);
    if (ts == 64) hipLaunchKernelGGL((sandwich_bwd_kernel<TX, TR, 64, WHOLE, GROUPS>), grid, block, 0, s, q, plan);
    else if (ts == 128) hipLaunchKernelGGL((sandwich_bwd_kernel<TX, TR, 128, WHOLE, GROUPS>), grid, block, 0, s, q, plan);
    else if (ts == 256) hipLaunchKernelGGL((sandwich_bwd_kernel<TX, TR, 256, WHOLE, GROUPS>), grid, block, 0, s, q, plan);
    else if (ts == 512) hipLaunchKernelGGL((sandwich_bwd_kernel<TX, TR, 512, WHOLE, GROUPS>), grid, block, 0, s, q, plan);
    else hipLaunchKernelGGL((sandwich_bwd_kernel<TX, TR, 1024, WHOLE, GROUPS>), grid, block, 0, s, q, plan);
}
template <typename TX, typename TR, bool WHOLE>
static int bwd_launch(const vms_sandwich_norm_bwd_params& q, hipStream_t s) {
    const vms_sandwich_norm_params& p = q.f;
    const Plan plan = plan_of(p);
    if (plan.whole) bwd_team<TX, TR, WHOLE, true>(q, plan, s);
    else bwd_team<TX, TR, WHOLE, false>(q, plan, s);
    VMS_LAUNCH_CHECK();
    const bool shared = p.gate && p.rows_per_gate > 1 && !plan.whole;   // gate rows that collect sums over workgroups
    hipLaunchKernelGGL(sandwich_finish_kernel, dim3((p.cols + 63) / 64, 4 + (shared ? plan.groups : 0)), dim3(1024), 0, s, q, plan, shared ? 1 : 0);
    VMS_LAUNCH_CHECK();
    return VMS_OK;
}

#define VMS_SN_TYPES(FN, TX, TR, P_, ARG, s)                                                                                             \
    (((P_).cols % 8 == 0) ? FN<TX, TR, true>(ARG, s) : FN<TX, TR, false>(ARG, s))
#define VMS_SN_DISPATCH(FN, P_, ARG, s)                                                                                                  \
    do {                                                                                                                                 \
        const bool f32_ = (P_).res_dtype == VMS_F32;                                                                                     \
        switch ((P_).x_dtype) {                                                                                                          \
            case VMS_F32: rc = VMS_SN_TYPES(FN, float, float, P_, ARG, s); break;                                                        \
            case VMS_F16: rc = f32_ ? VMS_SN_TYPES(FN, f16_t, float, P_, ARG, s) : VMS_SN_TYPES(FN, f16_t, f16_t, P_, ARG, s); break;    \
            default: rc = f32_ ? VMS_SN_TYPES(FN, bf16_t, float, P_, ARG, s) : VMS_SN_TYPES(FN, bf16_t, bf16_t, P_, ARG, s);             \
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
    if (!pp || pp->rows <= 0 || pp->cols <= 0 || pp->cols > 8192 || (pp->gate && (pp->rows_per_gate < 1 || pp->rows % pp->rows_per_gate != 0)))
        return 0;
    return (int64_t)sn::plan_of(*pp).partials * 4 * pp->cols * 4;
}
extern "C" int vms_sandwich_norm_bwd(const vms_sandwich_norm_bwd_params* qq, void* stream) {
    VMS_CHECK(qq != nullptr, "null params");
    const vms_sandwich_norm_bwd_params& q = *qq;
    if (int rc = sn::validate(q.f)) return rc;
    VMS_CHECK(q.f.stats && q.dx && q.dpost_weight && q.dpre_weight, "stats, dx, dpost_weight, dpre_weight are required");
    VMS_CHECK(!q.f.gate || q.dgate, "dgate comes with gate");
    VMS_CHECK(aligned16(q.workspace), "workspace must be 16-byte aligned");
    VMS_CHECK(q.workspace && q.workspace_bytes >= vms_sandwich_norm_bwd_workspace_bytes(&q.f), "workspace is too small (vms_sandwich_norm_bwd_workspace_bytes)");
    int rc = VMS_OK;
    VMS_SN_DISPATCH(sn::bwd_launch, q.f, q, static_cast<hipStream_t>(stream));
    if (rc == VMS_OK) set_last_kernel("sandwich_norm_bwd");
    return rc;
}
extern "C" int vms_sizeof_sandwich_norm_params(void) { return (int)sizeof(vms_sandwich_norm_params); }
extern "C" int vms_sizeof_sandwich_norm_bwd_params(void) { return (int)sizeof(vms_sandwich_norm_bwd_params); }
