// gated_delta_bwd.hip -- gated delta rule, backward (vms_gated_delta_bwd); algebra, precision and layouts: gated_delta.h.
//
// With S0, U, T, M of every chunk from the forward's workspace and dS1 = the adjoint of a chunk's last state:
//   gd_bwd_scan  walks the chunks from the end, a wave per 16 CT columns of dS as in the forward:
//                  dU = M^T dO + del K dS1;  Y = T^T dU;  dV = beta Y;  dS0 = gam_63 dS1 + Q^T (scale gam dO) - K^T (beta gam Y)
//                and leaves dS1 and Y
//   gd_grad      one workgroup per chunk and q / k head, no order among them:
//                  Z = Y U^T, DM = dO U^T (64 x 64);  dQ = scale (gam dO S0^T + (L DM) K)
//                  W = gam Y S0^T + (L Z, i > j) K      what k_i receives as the factor on the left is -beta_i W_i
//                  X = del U dS1^T + scale (L DM)^T Q + (-beta L Z, i > j)^T K     ... as the factor on the right
//                  dK = X - beta W;  dbeta_i = Y_i.V_i - k_i.W_i
//                  dG_i = q_i.dQ_i - beta_i k_i.W_i - k_i.X_i, and <S1, dS1> = gam_63 <S0, dS1> + sum_j del_j k_j.(U dS1^T)_j at the
//                  last token; dg = the sums of dG from a token to the chunk's end
//                No atomics: heads that share q / k are summed by the workgroup that owns the chunk, in order.
#include "gated_delta.h"

namespace vms {
namespace gd {

struct BwdArgs {   // what the kernels need of vms_gated_delta_bwd_params (one kernel argument block)
    vms_gated_delta_bwd_params q;
    Layout l;
};

// ---- the walk over the chunks, from the end ------------------------------------------------------------------
template <typename T, int KP, int NW, int CT>
__global__ __launch_bounds__(NW * 64, 1) void gd_bwd_scan_kernel(const BwdArgs a, const int slices) {
    constexpr int NX = Prec<T>::NX, NS = Prec<T>::NS, NO = Prec<T>::NO;
    constexpr int NT = NW * 64, KB = KP / 32, DT = KP / 16;
    constexpr int TB = tile_bytes<KP>();
    constexpr int PK = C * KP / 8 / NT;
    constexpr int PT = (768 * NS + NT - 1) / NT;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char* const Ks = lds;
    char* const Qs = Ks + NX * TB;
    char* const Ts = Qs + NX * TB;
    char* const Ms = Ts + NS * kTri;
    float* const gs = reinterpret_cast<float*>(Ms + NS * kTri);   // gam, bet, del

    const vms_gated_delta_params& p = a.q.f;
    const Layout& l = a.l;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, n = lane & 15, q4 = lane >> 4;
    int pair, slice;
    pair_of(blockIdx.x, p.batch * p.heads, slices, pair, slice);
    const int b = pair / p.heads, h = pair % p.heads, hk = h / (p.heads / p.heads_k);
    const int len = length_of(p, b), nc = (len + C - 1) / C;
    const int col0 = (slice * NW + w) * CT * 16;
    const bool active = col0 < l.vpad;
    const T* const qb = static_cast<const T*>(p.q) + (int64_t)b * p.q_batch_stride + (int64_t)hk * p.q_head_stride;
    const T* const kb_ = static_cast<const T*>(p.k) + (int64_t)b * p.k_batch_stride + (int64_t)hk * p.k_head_stride;
    const T* const dob = static_cast<const T*>(a.q.dout) + (int64_t)b * a.q.dout_batch_stride + (int64_t)h * a.q.dout_head_stride;
    const int64_t dv_seq = (int64_t)p.heads * p.dv;
    T* const dvb = static_cast<T*>(a.q.dv) + ((int64_t)b * p.seqlen * p.heads + h) * p.dv;
    const char* const ws = static_cast<const char*>(p.workspace);
    char* const wb = static_cast<char*>(a.q.workspace);
    const int64_t slot0 = (int64_t)pair * l.chunks;

    Raw8<T> kr[PK], qr[PK];
    bf16x8 tr[PT];
    float gr = 0.f;
    T vr[CT][4][4];
    auto fetch = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PK; ++i) {
            const int id = tid + i * NT, row = id / (KP / 8), cc = 8 * (id % (KP / 8)), at = c * C + row;
            const bool ok = at < len;
            const int64_t t = ok ? token(at, len, p.reverse) : 0;
            kr[i] = load_raw8<T>(kb_ + t * p.k_seq_stride, cc, p.dk, ok);
            qr[i] = load_raw8<T>(qb + t * p.q_seq_stride, cc, p.dk, ok);
        }
        const bf16x8* const t8 = reinterpret_cast<const bf16x8*>(ws + l.tri + (slot0 + c) * l.tri_slot);
#pragma unroll
        for (int i = 0; i < PT; ++i)
            if (tid + i * NT < 768 * NS) tr[i] = t8[tid + i * NT];
        const float* const g = reinterpret_cast<const float*>(reinterpret_cast<const Gates*>(ws + l.gates) + slot0 + c);
        if (tid < 3 * C) gr = g[tid];
        if (active) {
#pragma unroll
            for (int rt = 0; rt < 4; ++rt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = c * C + 16 * rt + 4 * q4 + r;
                    const bool ok = at < len;
                    const T* const row = dob + (ok ? (int64_t)token(at, len, p.reverse) * a.q.dout_seq_stride : 0);
#pragma unroll
                    for (int j = 0; j < CT; ++j) vr[j][rt][r] = ok && col0 + 16 * j + n < p.dv ? row[col0 + 16 * j + n] : static_cast<T>(0.f);
                }
        }
    };
    auto stage = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PK; ++i) {
            const int id = tid + i * NT, row = id / (KP / 8), cc = 8 * (id % (KP / 8));
            tile_put<KP, NX>(Ks, row, cc, planes_of<T>(kr[i]));
            tile_put<KP, NX>(Qs, row, cc, planes_of<T>(qr[i]));
        }
#pragma unroll
        for (int i = 0; i < PT; ++i)
            if (tid + i * NT < 768 * NS) reinterpret_cast<bf16x8*>(Ts)[tid + i * NT] = tr[i];
        if (tid < 3 * C) gs[tid] = gr;
    };

    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    f32x4 dS[DT][CT];
    const int64_t sbase = (int64_t)pair * p.dk * p.dv;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * d + 4 * q4 + r, col = col0 + 16 * j + n;
                dS[d][j][r] = a.q.dfinal_state && row < p.dk && col < p.dv ? a.q.dfinal_state[sbase + (int64_t)row * p.dv + col] : 0.f;
            }
    if (nc > 0) {
        fetch(nc - 1);
        stage();
    }
    for (int c = nc - 1; c >= 0; --c) {
        __syncthreads();
        f32x4 D[4][CT];   // dO
#pragma unroll
        for (int rt = 0; rt < 4; ++rt)
#pragma unroll
            for (int j = 0; j < CT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) D[rt][j][r] = static_cast<float>(vr[j][rt][r]);
        if (c > 0) fetch(c - 1);
        if (active) {
            const int64_t slot = slot0 + c;
            f32x4 dU[4][CT], Y[4][CT];
#pragma unroll
            for (int rt = 0; rt < 4; ++rt)
#pragma unroll
                for (int j = 0; j < CT; ++j) { dU[rt][j] = zero; Y[rt][j] = zero; }
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                Frag<NS> sf[CT];
#pragma unroll
                for (int j = 0; j < CT; ++j) {
                    sf[j] = frag_of<NS>(dS[2 * kb][j], dS[2 * kb + 1][j]);
                    if (col0 + 16 * j < l.vpad)
#pragma unroll
                        for (int half = 0; half < 2; ++half)
#pragma unroll
                            for (int i = 0; i < NO; ++i) {
                                const f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sf[j].p[i], unit_frag(half, n, q4), zero, 0, 0, 0);
                                store_planes4(wb + l.dS + slot * l.s_slot + 2 * (((int64_t)i * KP + 32 * kb + 16 * half + n) * l.vpad + col0 + 16 * j + 4 * q4), x);
                            }
                }
#pragma unroll
                for (int rt = 0; rt < 4; ++rt) {
                    const Frag<NX> kf = tile_rows<KP, NX>(Ks, rt, kb, n, q4);
#pragma unroll
                    for (int j = 0; j < CT; ++j) mma<NS>(dU[rt][j], kf, sf[j]);
                }
            }
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) {
                const f32x4 de = *reinterpret_cast<const f32x4*>(&gs[2 * C + 16 * rt + 4 * q4]);
#pragma unroll
                for (int j = 0; j < CT; ++j) dU[rt][j] *= de;
            }
#pragma unroll
            for (int ib = 0; ib < 2; ++ib) {
                Frag<NX> df[CT];
#pragma unroll
                for (int j = 0; j < CT; ++j) df[j] = frag_of<NX>(D[2 * ib][j], D[2 * ib + 1][j]);
#pragma unroll
                for (int ct = 0; ct < 2 * ib + 2; ++ct) {
                    const Frag<NS> mf = tri_cols<NS>(Ms, ct, ib, n, q4);
#pragma unroll
                    for (int j = 0; j < CT; ++j) mma<NS>(dU[ct][j], mf, df[j]);
                }
            }
#pragma unroll
            for (int ib = 0; ib < 2; ++ib) {
                Frag<NS> uf[CT];
#pragma unroll
                for (int j = 0; j < CT; ++j) uf[j] = frag_of<NS>(dU[2 * ib][j], dU[2 * ib + 1][j]);
#pragma unroll
                for (int ct = 0; ct < 2 * ib + 2; ++ct) {
                    const Frag<NS> tf = tri_cols<NS>(Ts, ct, ib, n, q4);
#pragma unroll
                    for (int j = 0; j < CT; ++j) mma<NS>(Y[ct][j], tf, uf[j]);
                }
            }
            const float glast = gs[C - 1];
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int j = 0; j < CT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) dS[d][j][r] *= glast;
#pragma unroll
            for (int ib = 0; ib < 2; ++ib) {
                const f32x4 g0 = *reinterpret_cast<const f32x4*>(&gs[32 * ib + 4 * q4]), g1 = *reinterpret_cast<const f32x4*>(&gs[32 * ib + 16 + 4 * q4]);
                const f32x4 b0 = *reinterpret_cast<const f32x4*>(&gs[C + 32 * ib + 4 * q4]), b1 = *reinterpret_cast<const f32x4*>(&gs[C + 32 * ib + 16 + 4 * q4]);
                Frag<NS> qf[CT], yf[CT];
#pragma unroll
                for (int j = 0; j < CT; ++j) {
                    f32x4 x0, x1, y0, y1;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x0[r] = p.scale * g0[r] * D[2 * ib][j][r];
                        x1[r] = p.scale * g1[r] * D[2 * ib + 1][j][r];
                        y0[r] = b0[r] * Y[2 * ib][j][r];
                        y1[r] = b1[r] * Y[2 * ib + 1][j][r];
                    }
                    qf[j] = frag_of<NS>(x0, x1);
                    if (col0 + 16 * j < l.vpad) {   // Y for gd_grad, dV = beta Y
                        const Frag<NO> yo = frag_of<NO>(Y[2 * ib][j], Y[2 * ib + 1][j]), vo = frag_of<NO>(y0, y1);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const bf16x8 one = unit_frag(half, n, q4);
                            f32x4 dv = zero;
#pragma unroll
                            for (int i = NO - 1; i >= 0; --i) {
                                const f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(yo.p[i], one, zero, 0, 0, 0);
                                store_planes4(wb + l.Y + slot * l.u_slot + 2 * (((int64_t)i * C + 32 * ib + 16 * half + n) * l.vpad + col0 + 16 * j + 4 * q4), x);
                                dv = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo.p[i], one, dv, 0, 0, 0);
                            }
                            const int at = c * C + 32 * ib + 16 * half + n;
                            if (at < len) store4<T>(dvb + (int64_t)token(at, len, p.reverse) * dv_seq, col0 + 16 * j + 4 * q4, p.dv, dv);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) { y0[r] *= -g0[r]; y1[r] *= -g1[r]; }
                    yf[j] = frag_of<NS>(y0, y1);
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const Frag<NX> qc = tile_cols<KP, NX>(Qs, d, ib, n, q4), kc = tile_cols<KP, NX>(Ks, d, ib, n, q4);
#pragma unroll
                    for (int j = 0; j < CT; ++j) {
                        mma<NS>(dS[d][j], qc, qf[j]);
                        mma<NS>(dS[d][j], kc, yf[j]);
                    }
                }
            }
        }
        __syncthreads();
        if (c > 0) stage();
    }
    if (active && a.q.dinitial_state) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int j = 0; j < CT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * d + 4 * q4 + r, col = col0 + 16 * j + n;
                    if (row < p.dk && col < p.dv) a.q.dinitial_state[sbase + (int64_t)row * p.dv + col] = dS[d][j][r];
                }
    }
    const int c0 = slice * NW * CT * 16, cn = (p.dv - c0) < NW * CT * 16 ? (p.dv - c0) : NW * CT * 16;
    for (int t = len + w; t < p.seqlen; t += NW)
        for (int cc = lane; cc < cn; cc += 64) dvb[(int64_t)t * dv_seq + c0 + cc] = static_cast<T>(0.f);
}

// ---- dq, dk, dg, dbeta of one chunk --------------------------------------------------------------------------
__device__ __forceinline__ void st_gate(void* p, int64_t i, int dt, float v) {
    if (dt == VMS_F32) static_cast<float*>(p)[i] = v;
    else if (dt == VMS_F16) static_cast<f16_t*>(p)[i] = static_cast<f16_t>(v);
    else static_cast<bf16_t*>(p)[i] = static_cast<bf16_t>(v);
}
__device__ __forceinline__ float quarters_sum(float v) {   // over the four lanes 16 q + n
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float L_of(double d) { return fast_exp2((float)(d * 1.4426950408889634)); }

template <typename T, int KP>
__global__ __launch_bounds__(256, 1) void gd_grad_kernel(const BwdArgs a) {
    constexpr int NX = Prec<T>::NX, NS = Prec<T>::NS, NO = Prec<T>::NO, DT = KP / 16, TB = tile_bytes<KP>();
    constexpr int PK = C * KP / 8 / 256;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char* const Ks = lds;
    char* const Qs = Ks + NX * TB;
    Gates* const gs = reinterpret_cast<Gates*>(Qs + NX * TB);
    float* const dGs = reinterpret_cast<float*>(gs + 1);
    float* const part = dGs + C;   // one sum per wave

    const vms_gated_delta_params& p = a.q.f;
    const Layout& l = a.l;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, q4 = lane >> 4;
    const int c = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
    const int rep = p.heads / p.heads_k;
    const int len = length_of(p, b);
    const int64_t dk_seq = (int64_t)p.heads_k * p.dk;
    T* const dqb = static_cast<T*>(a.q.dq) + ((int64_t)b * p.seqlen * p.heads_k + hk) * p.dk;
    T* const dkb = static_cast<T*>(a.q.dk) + ((int64_t)b * p.seqlen * p.heads_k + hk) * p.dk;

    // padding rows of this chunk
    {
        const int first = c * C > len ? c * C : len, end = (c + 1) * C < p.seqlen ? (c + 1) * C : p.seqlen;
        for (int t = first + w; t < end; t += 4) {
            for (int cc = lane; cc < p.dk; cc += 64) {
                dqb[(int64_t)t * dk_seq + cc] = static_cast<T>(0.f);
                dkb[(int64_t)t * dk_seq + cc] = static_cast<T>(0.f);
            }
            for (int r = lane; r < rep; r += 64) {
                const int64_t at = ((int64_t)b * p.seqlen + t) * p.heads + hk * rep + r;
                st_gate(a.q.dg, at, p.gate_dtype, 0.f);
                st_gate(a.q.dbeta, at, p.gate_dtype, 0.f);
            }
        }
    }
    if (c * C >= len) return;

    const T* const qb = static_cast<const T*>(p.q) + (int64_t)b * p.q_batch_stride + (int64_t)hk * p.q_head_stride;
    const T* const kb_ = static_cast<const T*>(p.k) + (int64_t)b * p.k_batch_stride + (int64_t)hk * p.k_head_stride;
#pragma unroll
    for (int i = 0; i < PK; ++i) {
        const int id = tid + i * 256, row = id / (KP / 8), cc = 8 * (id % (KP / 8)), at = c * C + row;
        const bool ok = at < len;
        const int64_t t = ok ? token(at, len, p.reverse) : 0;
        tile_put<KP, NX>(Ks, row, cc, planes_of<T>(load_raw8<T>(kb_ + t * p.k_seq_stride, cc, p.dk, ok)));
        tile_put<KP, NX>(Qs, row, cc, planes_of<T>(load_raw8<T>(qb + t * p.q_seq_stride, cc, p.dk, ok)));
    }
    const char* const ws = static_cast<const char*>(p.workspace);
    const char* const wb = static_cast<const char*>(a.q.workspace);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const int own = 16 * w + n, at_own = c * C + own;   // this lane's token
    const bool ok_own = at_own < len;
    f32x4 dqs[DT], dks[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) { dqs[d] = zero; dks[d] = zero; }

    for (int r = 0; r < rep; ++r) {
        const int h = hk * rep + r;
        const int64_t slot = ((int64_t)b * p.heads + h) * l.chunks + c;
        __syncthreads();   // the tiles are there / the previous head's gates are no longer read
        {
            const float* const src = reinterpret_cast<const float*>(reinterpret_cast<const Gates*>(ws + l.gates) + slot);
            for (int i = tid; i < (int)(sizeof(Gates) / 4); i += 256) reinterpret_cast<float*>(gs)[i] = src[i];
        }
        const char* const Uw = ws + l.U + slot * l.u_slot;
        const char* const Yw = wb + l.Y + slot * l.u_slot;
        const char* const Sw = ws + l.S0 + slot * l.s_slot;
        const char* const Dw = wb + l.dS + slot * l.s_slot;
        const T* const vb = static_cast<const T*>(p.v) + (int64_t)b * p.v_batch_stride + (int64_t)h * p.v_head_stride;
        const T* const dob = static_cast<const T*>(a.q.dout) + (int64_t)b * a.q.dout_batch_stride + (int64_t)h * a.q.dout_head_stride;
        auto planes = [&](const char* base, int rows, int row, int vblk) __attribute__((always_inline)) {   // natural order: 8 columns from 32 vblk + 8 q4
            Frag<NO> f;
#pragma unroll
            for (int i = 0; i < NO; ++i)
                f.p[i] = *reinterpret_cast<const bf16x8*>(base + 2 * (((int64_t)i * rows + row) * l.vpad + 32 * vblk + 8 * q4));
            return f;
        };
        auto out_rows = [&](int tok, int vblk) __attribute__((always_inline)) {
            const int at = c * C + tok;
            const bool ok = at < len;
            return planes_of<T>(load_raw8<T>(dob + (ok ? (int64_t)token(at, len, p.reverse) * a.q.dout_seq_stride : 0), 32 * vblk + 8 * q4, p.dv, ok));
        };
        // [j][i]: rows = another tile's tokens, columns (lanes) = this wave's tokens
        f32x4 dm[4], zl[4];   // this wave's tokens as i, tiles j <= w: dO_i.U_j, Y_i.U_j
        f32x4 mt[4], zr[4];   // this wave's tokens as j, tiles i >= w
        f32x4 OS[DT], YS[DT], US[DT];
#pragma unroll
        for (int t = 0; t < 4; ++t) { dm[t] = zero; zl[t] = zero; mt[t] = zero; zr[t] = zero; }
#pragma unroll
        for (int d = 0; d < DT; ++d) { OS[d] = zero; YS[d] = zero; US[d] = zero; }
        float yv = 0.f, ss = 0.f;
        for (int vk = 0; vk < l.vpad / 32; ++vk) {
            const Frag<NO> yi = planes(Yw, C, own, vk), ui = planes(Uw, C, own, vk);
            const Frag<NX> oi = out_rows(own, vk);
            {
                const Raw8<T> v = load_raw8<T>(vb + (ok_own ? (int64_t)token(at_own, len, p.reverse) * p.v_seq_stride : 0), 32 * vk + 8 * q4, p.dv, ok_own);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float y = 0.f;
#pragma unroll
                    for (int i = NO - 1; i >= 0; --i) y += static_cast<float>(yi.p[i][e]);
                    yv = fmaf(y, static_cast<float>(v.v[e]), yv);
                }
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (t <= w) {
                    const Frag<NO> uj = planes(Uw, C, 16 * t + n, vk);
                    mma<NO>(dm[t], uj, oi);
                    mma<NO>(zl[t], uj, yi);
                }
                if (t >= w) {
                    mma<NO>(mt[t], out_rows(16 * t + n, vk), ui);
                    mma<NO>(zr[t], planes(Yw, C, 16 * t + n, vk), ui);
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const Frag<NO> s0 = planes(Sw, KP, 16 * d + n, vk), s1 = planes(Dw, KP, 16 * d + n, vk);
                mma<NO>(OS[d], s0, oi);
                mma<NO>(YS[d], s0, yi);
                mma<NO>(US[d], s1, ui);
                if ((d & 3) == w) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float x = 0.f, y = 0.f;
#pragma unroll
                        for (int i = NO - 1; i >= 0; --i) { x += static_cast<float>(s0.p[i][e]); y += static_cast<float>(s1.p[i][e]); }
                        ss = fmaf(x, y, ss);
                    }
                }
            }
        }
        __syncthreads();   // gates
        const float gi = gs->gam[own], di = gs->del[own], bi = gs->bet[own];
        const double Gi = gs->G[own];
        float ku = 0.f;
        auto rowdot = [&](const char* tile, const f32x4 (&x)[DT]) __attribute__((always_inline)) {
            float s = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                f32x4 v = zero;
#pragma unroll
                for (int i = NX - 1; i >= 0; --i) {
                    const bf16x4 t4 = *reinterpret_cast<const bf16x4*>(tile + i * TB + own * tile_row<KP>() + 2 * (32 * (d >> 1) + 8 * q4 + 4 * (d & 1)));
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += static_cast<float>(t4[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s = fmaf(v[e], x[d][e], s);
            }
            return s;
        };
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                OS[d][e] *= p.scale * gi;
                YS[d][e] *= gi;
                US[d][e] *= di;
            }
        ku = rowdot(Ks, US);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int o = 16 * t + 4 * q4 + e;
                const double Go = gs->G[o];
                if (t <= w) {   // o = j
                    const float L = o <= own ? L_of(Gi - Go) : 0.f;
                    dm[t][e] *= p.scale * L;
                    zl[t][e] = o < own ? L * zl[t][e] : 0.f;
                }
                if (t >= w) {   // o = i
                    const float L = o >= own ? L_of(Go - Gi) : 0.f;
                    mt[t][e] *= p.scale * L;
                    zr[t][e] = o > own ? -gs->bet[o] * L * zr[t][e] : 0.f;
                }
            }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            if (2 * kb <= w) {
                const Frag<NS> fm = frag_of<NS>(dm[2 * kb], dm[2 * kb + 1]), fz = frag_of<NS>(zl[2 * kb], zl[2 * kb + 1]);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const Frag<NX> kc = tile_cols<KP, NX>(Ks, d, kb, n, q4);
                    mma<NS>(OS[d], kc, fm);
                    mma<NS>(YS[d], kc, fz);
                }
            }
            if (2 * kb + 1 >= w) {
                const Frag<NS> fm = frag_of<NS>(mt[2 * kb], mt[2 * kb + 1]), fz = frag_of<NS>(zr[2 * kb], zr[2 * kb + 1]);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    mma<NS>(US[d], tile_cols<KP, NX>(Qs, d, kb, n, q4), fm);
                    mma<NS>(US[d], tile_cols<KP, NX>(Ks, d, kb, n, q4), fz);
                }
            }
        }
        const float qd = quarters_sum(rowdot(Qs, OS)), kw = quarters_sum(rowdot(Ks, YS)), kx = quarters_sum(rowdot(Ks, US));
        yv = quarters_sum(yv);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                dqs[d][e] += OS[d][e];
                dks[d][e] += US[d][e] - bi * YS[d][e];
            }
        const int64_t gate_at = ok_own ? ((int64_t)b * p.seqlen + token(at_own, len, p.reverse)) * p.heads + h : 0;
        if (q4 == 0) {
            dGs[own] = qd - bi * kw - kx;
            if (ok_own) st_gate(a.q.dbeta, gate_at, p.gate_dtype, yv - kw);
        }
        ss = wave_sum(gs->gam[C - 1] * ss + ku);
        if (lane == 0) part[w] = ss;
        __syncthreads();
        if (w == 0) {   // lane = token
            float x = dGs[lane];
#pragma unroll
            for (int s = 1; s < 64; s *= 2) {
                const float o = __shfl_down(x, s);
                if (lane + s < 64) x += o;
            }
            x += part[0] + part[1] + part[2] + part[3];
            const int at = c * C + lane;
            if (at < len) st_gate(a.q.dg, ((int64_t)b * p.seqlen + token(at, len, p.reverse)) * p.heads + h, p.gate_dtype, x);
        }
    }
    if (ok_own) {
        const int64_t t = token(at_own, len, p.reverse);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            store4<T>(dqb + t * dk_seq, 16 * d + 4 * q4, p.dk, dqs[d]);
            store4<T>(dkb + t * dk_seq, 16 * d + 4 * q4, p.dk, dks[d]);
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------
static int allow_lds(PerDeviceOnce& once, const void* kernel, int bytes) {
    if (bytes <= 65536) return VMS_OK;
    const hipError_t e = once.run([&] { return hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes); });
    if (e != hipSuccess) { set_error("hipFuncSetAttribute: %s", hipGetErrorString(e)); return VMS_ERR_LAUNCH; }
    return VMS_OK;
}
template <typename T, int KP, int NW, int CT>
static int bwd_scan_launch(const BwdArgs& a, hipStream_t s) {
    constexpr int NX = Prec<T>::NX, NS = Prec<T>::NS;
    constexpr int lds = 2 * NX * tile_bytes<KP>() + 2 * NS * kTri + 3 * C * 4;
    static_assert(NW * 64 >= 3 * C && lds <= 163840, "a thread per gate; 160 KB of LDS");
    static PerDeviceOnce once;
    if (int rc = allow_lds(once, reinterpret_cast<const void*>(&gd_bwd_scan_kernel<T, KP, NW, CT>), lds)) return rc;
    const int slices = (a.l.vpad + NW * CT * 16 - 1) / (NW * CT * 16);
    hipLaunchKernelGGL((gd_bwd_scan_kernel<T, KP, NW, CT>), dim3(a.q.f.batch * a.q.f.heads * slices), dim3(NW * 64), lds, s, a, slices);
    VMS_LAUNCH_CHECK();
    return VMS_OK;
}
template <typename T, int KP>
static int bwd_launch(const BwdArgs& a, hipStream_t s) {
    if (int rc = bwd_scan_launch<T, KP, 4, 1>(a, s)) return rc;
    constexpr int lds = 2 * Prec<T>::NX * tile_bytes<KP>() + (int)sizeof(Gates) + (C + 4) * 4;
    static PerDeviceOnce once;
    if (int rc = allow_lds(once, reinterpret_cast<const void*>(&gd_grad_kernel<T, KP>), lds)) return rc;
    hipLaunchKernelGGL((gd_grad_kernel<T, KP>), dim3(a.l.chunks, a.q.f.heads_k, a.q.f.batch), dim3(256), lds, s, a);
    VMS_LAUNCH_CHECK();
    return VMS_OK;
}
template <typename T>
static int bwd_type(const BwdArgs& a, hipStream_t s) {
    return pad_k(a.q.f.dk) == 64 ? bwd_launch<T, 64>(a, s) : bwd_launch<T, 128>(a, s);
}

}  // namespace gd
}  // namespace vms

using namespace vms;

extern "C" int vms_gated_delta_bwd(const vms_gated_delta_bwd_params* qq, void* stream) {
    VMS_CHECK(qq != nullptr, "null params");
    if (int rc = gd::validate(qq->f)) return rc;
    VMS_CHECK(qq->f.for_backward, "the forward must have run with for_backward");
    VMS_CHECK(qq->dout && qq->dq && qq->dk && qq->dv && qq->dg && qq->dbeta, "dout, dq, dk, dv, dg, dbeta are required");
    gd::BwdArgs a{*qq, gd::layout(qq->f)};
    VMS_CHECK(qq->workspace != nullptr && qq->workspace_bytes >= a.l.bwd_bytes, "workspace is too small (vms_gated_delta_bwd_workspace_bytes)");
    VMS_CHECK((reinterpret_cast<uintptr_t>(qq->workspace) & 15) == 0, "workspace must be 16-byte aligned");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int dt = qq->f.dtype;
    const int rc = dt == VMS_BF16 ? gd::bwd_type<bf16_t>(a, s) : dt == VMS_F16 ? gd::bwd_type<f16_t>(a, s) : gd::bwd_type<float>(a, s);
    if (rc == VMS_OK) set_last_kernel("gated_delta_bwd");
    return rc;
}
extern "C" int vms_sizeof_gated_delta_bwd_params(void) { return (int)sizeof(vms_gated_delta_bwd_params); }
