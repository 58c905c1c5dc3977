// gated_delta_fwd.hip -- gated delta rule, forward (vms_gated_delta_fwd): the algebra and the layouts are in gated_delta.h.
//
//   gd_prep   one wave per (chunk, head): the gates, T (triangular inverse in fp32), M.
//   gd_scan   the walk over the chunks.  The columns of S (and of V, U, O) never meet: a wave owns 16 CT of them for the whole
//             sequence, S in its accumulators, and shares only the operands K, Q, T, M of a chunk with the other waves of its
//             workgroup through LDS.
#include "gated_delta.h"

namespace vms {
namespace gd {

// g below this forgets everything (exp underflows) and would cost the cumulative sums their low bits
constexpr float kMinGate = -104.f;

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// ---- T, M and gates of one chunk -----------------------------------------------------------------------------
// K K^T and Q K^T (16x16x32 bf16 MFMA, operands straight from memory), L from double cumulative sums (differences of long sums keep
// their bits), then T: the four 16 x 16 diagonal blocks by forward substitution (16 lanes each, a column per lane; a power series would
// lose ~13 bits to the binomials of equal keys), joined by T21 = -T22 A21 T11 with fp32 MFMA.
template <typename T, int KP>
__global__ __launch_bounds__(64, 2) void gd_prep_kernel(const vms_gated_delta_params p, const Layout l) {
    constexpr int NX = Prec<T>::NX, NS = Prec<T>::NS;
    constexpr int AR = 68;   // row pitch of As, floats
    __shared__ __attribute__((aligned(16))) float As[C * AR];
    __shared__ double Gs[C];
    __shared__ float bs[C];
    const int lane = threadIdx.x, n = lane & 15, q4 = lane >> 4;
    const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int len = length_of(p, b);
    if (c * C >= len) return;
    const int hk = h / (p.heads / p.heads_k);
    const int64_t slot = ((int64_t)b * p.heads + h) * l.chunks + c;
    char* const ws = static_cast<char*>(p.workspace);

    {   // gates: lane = token
        const int i = c * C + lane;
        float g = 0.f, be = 0.f;
        if (i < len) {
            const int64_t t = token(i, len, p.reverse);
            g = ld_gate(p.g, (int64_t)b * p.g_batch_stride + t * p.g_seq_stride + (int64_t)h * p.g_head_stride, p.gate_dtype);
            be = ld_gate(p.beta, (int64_t)b * p.beta_batch_stride + t * p.beta_seq_stride + (int64_t)h * p.beta_head_stride, p.gate_dtype);
            g = g < kMinGate ? kMinGate : g;
        }
        double G = g;
#pragma unroll
        for (int s = 1; s < 64; s *= 2) {
            const double o = __shfl_up(G, s);
            if (lane >= s) G += o;
        }
        const double last = __shfl(G, 63);
        Gs[lane] = G;
        bs[lane] = be;
        Gates* const o = reinterpret_cast<Gates*>(ws + l.gates) + slot;
        o->gam[lane] = fast_exp2((float)(G * 1.4426950408889634));
        o->bet[lane] = be;
        o->del[lane] = fast_exp2((float)((last - G) * 1.4426950408889634));
        o->G[lane] = G;
    }
    __syncthreads();

    const T* const qb = static_cast<const T*>(p.q) + (int64_t)b * p.q_batch_stride + (int64_t)hk * p.q_head_stride;
    const T* const kb_ = static_cast<const T*>(p.k) + (int64_t)b * p.k_batch_stride + (int64_t)hk * p.k_head_stride;
    auto rows = [&](const T* base, int64_t stride, int rt, int kb) {
        const int i = c * C + 16 * rt + n;
        const bool ok = i < len;
        return planes_of<T>(load_raw8<T>(base + (ok ? (int64_t)token(i, len, p.reverse) * stride : 0), 32 * kb + 8 * q4, p.dk, ok));
    };
    char* const tw = ws + l.tri + slot * l.tri_slot;
    char* const mw = tw + NS * kTri;
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
        f32x4 kk[4], qk[4];
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) { kk[ct] = f32x4{0.f, 0.f, 0.f, 0.f}; qk[ct] = f32x4{0.f, 0.f, 0.f, 0.f}; }
#pragma unroll
        for (int kb = 0; kb < KP / 32; ++kb) {
            const Frag<NX> qi = rows(qb, p.q_seq_stride, rt, kb), ki = rows(kb_, p.k_seq_stride, rt, kb);
#pragma unroll
            for (int ct = 0; ct <= rt; ++ct) {   // [j][i]: lane i, 4 consecutive j
                const Frag<NX> kj = ct == rt ? ki : rows(kb_, p.k_seq_stride, ct, kb);
                mma<NS>(kk[ct], kj, ki);
                mma<NS>(qk[ct], kj, qi);
            }
        }
        const int i = 16 * rt + n;
        const double Gi = Gs[i];
        const float bi = bs[i];
#pragma unroll
        for (int ct = 0; ct <= rt; ++ct) {
            f32x4 a;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = 16 * ct + 4 * q4 + r;
                const float L = j <= i ? fast_exp2((float)((Gi - Gs[j]) * 1.4426950408889634)) : 0.f;
                a[r] = j < i ? bi * L * kk[ct][r] : 0.f;
                qk[ct][r] = j <= i ? p.scale * L * qk[ct][r] : 0.f;
            }
            *reinterpret_cast<f32x4*>(&As[i * AR + 16 * ct + 4 * q4]) = a;
        }
#pragma unroll
        for (int kb = 0; kb <= rt / 2; ++kb) {
            const Frag<NS> f = frag_of<NS>(qk[2 * kb], qk[2 * kb + 1]);
#pragma unroll
            for (int i2 = 0; i2 < NS; ++i2)
                *reinterpret_cast<bf16x8*>(mw + i2 * kTri + 1024 * tri(rt, kb) + 16 * lane) = f.p[i2];
        }
    }
    __syncthreads();

    {   // diagonal blocks: quarter q4 inverts block q4, lane n its column n
        float t[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float acc = i == n ? 1.f : 0.f;
#pragma unroll
            for (int j4 = 0; j4 < (i + 3) / 4; ++j4) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(&As[(16 * q4 + i) * AR + 16 * q4 + 4 * j4]);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (4 * j4 + r < i) acc = fmaf(-a[r], t[4 * j4 + r], acc);
            }
            t[i] = acc;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) As[(16 * q4 + i) * AR + 16 * q4 + n] = t[i];
    }
    __syncthreads();
    // X += A[R][m] B[m][Cc]: the 16 x 16 block (R, m) of As times a block held as accumulator registers or in As
    auto a_of = [&](int R, int m) { return *reinterpret_cast<const f32x4*>(&As[(16 * R + n) * AR + 16 * m + 4 * q4]); };
    auto b_of = [&](int m, int Cc) {
        f32x4 v;
#pragma unroll
        for (int s = 0; s < 4; ++s) v[s] = As[(16 * m + 4 * q4 + s) * AR + 16 * Cc + n];
        return v;
    };
    auto mul = [&](f32x4& acc, const f32x4& a, const f32x4& b) {
#pragma unroll
        for (int s = 0; s < 4; ++s) acc = mfma4(a[s], b[s], acc);
    };
    auto put = [&](int R, int Cc, const f32x4& v) {
#pragma unroll
        for (int s = 0; s < 4; ++s) As[(16 * R + 4 * q4 + s) * AR + 16 * Cc + n] = -v[s];
    };
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    {
        f32x4 x0 = zero, x1 = zero, y0 = zero, y1 = zero;
        mul(x0, a_of(1, 0), b_of(0, 0));
        mul(x1, a_of(3, 2), b_of(2, 2));
        mul(y0, a_of(1, 1), x0);
        mul(y1, a_of(3, 3), x1);
        __syncthreads();
        put(1, 0, y0);
        put(3, 2, y1);
    }
    __syncthreads();
    {
        f32x4 x[2][2], y[2][2];
#pragma unroll
        for (int R = 0; R < 2; ++R) {
            x[R][0] = zero; x[R][1] = zero; y[R][0] = zero; y[R][1] = zero;
            mul(x[R][0], a_of(2 + R, 0), b_of(0, 0));
            mul(x[R][0], a_of(2 + R, 1), b_of(1, 0));
            mul(x[R][1], a_of(2 + R, 1), b_of(1, 1));
        }
#pragma unroll
        for (int Cc = 0; Cc < 2; ++Cc) {
            mul(y[0][Cc], a_of(2, 2), x[0][Cc]);
            mul(y[1][Cc], a_of(3, 2), x[0][Cc]);
            mul(y[1][Cc], a_of(3, 3), x[1][Cc]);
        }
        __syncthreads();
#pragma unroll
        for (int R = 0; R < 2; ++R)
#pragma unroll
            for (int Cc = 0; Cc < 2; ++Cc) put(2 + R, Cc, y[R][Cc]);
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < 4; ++rt)
#pragma unroll
        for (int kb = 0; kb <= rt / 2; ++kb) {
            const f32x4 lo = a_of(rt, 2 * kb), hi = 2 * kb + 1 <= rt ? a_of(rt, 2 * kb + 1) : zero;
            const Frag<NS> f = frag_of<NS>(lo, hi);
#pragma unroll
            for (int i2 = 0; i2 < NS; ++i2) *reinterpret_cast<bf16x8*>(tw + i2 * kTri + 1024 * tri(rt, kb) + 16 * lane) = f.p[i2];
        }
}

// ---- the walk over the chunks --------------------------------------------------------------------------------
template <typename T, int KP, int NW, int CT>
__global__ __launch_bounds__(NW * 64, 1) void gd_scan_kernel(const vms_gated_delta_params p, const Layout l, const int slices) {
    constexpr int NX = Prec<T>::NX, NS = Prec<T>::NS, NO = Prec<T>::NO;
    constexpr int NT = NW * 64, KB = KP / 32, DT = KP / 16;
    constexpr int TB = tile_bytes<KP>();
    constexpr int PK = C * KP / 8 / NT;                       // 8-element pieces of a k / q tile per thread
    constexpr int PT = (768 * NS + NT - 1) / NT;              // 16-byte pieces of T and M per thread
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char* const Ks = lds;
    char* const Qs = Ks + NX * TB;
    char* const Ts = Qs + NX * TB;
    char* const Ms = Ts + NS * kTri;
    float* const gs = reinterpret_cast<float*>(Ms + NS * kTri);   // gam, bet, del

    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, n = lane & 15, q4 = lane >> 4;
    int pair, slice;
    pair_of(blockIdx.x, p.batch * p.heads, slices, pair, slice);
    const int b = pair / p.heads, h = pair % p.heads, hk = h / (p.heads / p.heads_k);
    const int len = length_of(p, b), nc = (len + C - 1) / C;
    const int col0 = (slice * NW + w) * CT * 16;
    const bool active = col0 < l.vpad;   // uniform in the wave
    const T* const qb = static_cast<const T*>(p.q) + (int64_t)b * p.q_batch_stride + (int64_t)hk * p.q_head_stride;
    const T* const kb_ = static_cast<const T*>(p.k) + (int64_t)b * p.k_batch_stride + (int64_t)hk * p.k_head_stride;
    const T* const vb = static_cast<const T*>(p.v) + (int64_t)b * p.v_batch_stride + (int64_t)h * p.v_head_stride;
    T* const ob = static_cast<T*>(p.out) + (int64_t)b * p.out_batch_stride + (int64_t)h * p.out_head_stride;
    char* const ws = static_cast<char*>(p.workspace);
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
                    const T* const row = vb + (ok ? (int64_t)token(at, len, p.reverse) * p.v_seq_stride : 0);
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
    f32x4 S[DT][CT];
    const int64_t sbase = (int64_t)pair * p.dk * p.dv;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * d + 4 * q4 + r, col = col0 + 16 * j + n;
                S[d][j][r] = p.initial_state && row < p.dk && col < p.dv ? p.initial_state[sbase + (int64_t)row * p.dv + col] : 0.f;
            }

    if (nc > 0) {
        fetch(0);
        stage();
    }
    for (int c = 0; c < nc; ++c) {
        __syncthreads();
        f32x4 R[4][CT];   // V of this chunk: its registers are the next chunk's from the fetch on
#pragma unroll
        for (int rt = 0; rt < 4; ++rt)
#pragma unroll
            for (int j = 0; j < CT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) R[rt][j][r] = static_cast<float>(vr[j][rt][r]);
        if (c + 1 < nc) fetch(c + 1);
        if (active) {
            f32x4 P[4][CT], O[4][CT];
#pragma unroll
            for (int rt = 0; rt < 4; ++rt)
#pragma unroll
                for (int j = 0; j < CT; ++j) { P[rt][j] = zero; O[rt][j] = zero; }
            const int64_t slot = slot0 + c;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                Frag<NS> sf[CT];
#pragma unroll
                for (int j = 0; j < CT; ++j) sf[j] = frag_of<NS>(S[2 * kb][j], S[2 * kb + 1][j]);
                if (p.for_backward) {   // S0 by rows (dk): 4 consecutive columns per lane
#pragma unroll
                    for (int j = 0; j < CT; ++j)
                        if (col0 + 16 * j < l.vpad)
#pragma unroll
                            for (int half = 0; half < 2; ++half)
#pragma unroll
                                for (int i = 0; i < NO; ++i) {
                                    const f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sf[j].p[i], unit_frag(half, n, q4), zero, 0, 0, 0);
                                    store_planes4(ws + l.S0 + slot * l.s_slot + 2 * (((int64_t)i * KP + 32 * kb + 16 * half + n) * l.vpad + col0 + 16 * j + 4 * q4), x);
                                }
                }
#pragma unroll
                for (int rt = 0; rt < 4; ++rt) {
                    const Frag<NX> kf = tile_rows<KP, NX>(Ks, rt, kb, n, q4), qf = tile_rows<KP, NX>(Qs, rt, kb, n, q4);
#pragma unroll
                    for (int j = 0; j < CT; ++j) {
                        mma<NS>(P[rt][j], kf, sf[j]);    // [token][v]
                        mma<NO>(O[rt][j], sf[j], qf);    // [v][token]: the lanes of a store hold 4 consecutive v
                    }
                }
            }
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) {
                const f32x4 ga = *reinterpret_cast<const f32x4*>(&gs[16 * rt + 4 * q4]), be = *reinterpret_cast<const f32x4*>(&gs[C + 16 * rt + 4 * q4]);
                const float sg = p.scale * gs[16 * rt + n];
#pragma unroll
                for (int j = 0; j < CT; ++j) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) R[rt][j][r] = be[r] * fmaf(-ga[r], P[rt][j][r], R[rt][j][r]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) O[rt][j][r] *= sg;
                }
            }
            f32x4 U[4][CT];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                Frag<NS> rf[CT];
#pragma unroll
                for (int j = 0; j < CT; ++j) rf[j] = frag_of<NS>(R[2 * kb][j], R[2 * kb + 1][j]);
#pragma unroll
                for (int rt = 2 * kb; rt < 4; ++rt) {
                    const Frag<NS> tf = tri_rows<NS>(Ts, rt, kb, lane);
#pragma unroll
                    for (int j = 0; j < CT; ++j) {
                        if (kb == 0) U[rt][j] = zero;
                        mma<NS>(U[rt][j], tf, rf[j]);
                    }
                }
            }
            const float glast = gs[C - 1];
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int j = 0; j < CT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[d][j][r] *= glast;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                Frag<NS> uf[CT];
#pragma unroll
                for (int j = 0; j < CT; ++j) {
                    const Frag<NS> of = frag_of<NS>(U[2 * kb][j], U[2 * kb + 1][j]);
#pragma unroll
                    for (int rt = 2 * kb; rt < 4; ++rt) mma<NS>(O[rt][j], of, tri_rows<NS>(Ms, rt, kb, lane));
                    if (p.for_backward && col0 + 16 * j < l.vpad) {
#pragma unroll
                        for (int half = 0; half < 2; ++half)
#pragma unroll
                            for (int i = 0; i < NO; ++i) {
                                const f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(of.p[i], unit_frag(half, n, q4), zero, 0, 0, 0);
                                store_planes4(ws + l.U + slot * l.u_slot + 2 * (((int64_t)i * C + 32 * kb + 16 * half + n) * l.vpad + col0 + 16 * j + 4 * q4), x);
                            }
                    }
                    f32x4 a = U[2 * kb][j], a2 = U[2 * kb + 1][j];
                    a *= *reinterpret_cast<const f32x4*>(&gs[2 * C + 32 * kb + 4 * q4]);
                    a2 *= *reinterpret_cast<const f32x4*>(&gs[2 * C + 32 * kb + 16 + 4 * q4]);
                    uf[j] = frag_of<NS>(a, a2);
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const Frag<NX> kf = tile_cols<KP, NX>(Ks, d, kb, n, q4);
#pragma unroll
                    for (int j = 0; j < CT; ++j) mma<NS>(S[d][j], kf, uf[j]);
                }
            }
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) {
                const int at = c * C + 16 * rt + n;
                if (at < len) {
                    T* const row = ob + (int64_t)token(at, len, p.reverse) * p.out_seq_stride;
#pragma unroll
                    for (int j = 0; j < CT; ++j) store4<T>(row, col0 + 16 * j + 4 * q4, p.dv, O[rt][j]);
                }
            }
        }
        __syncthreads();
        if (c + 1 < nc) stage();
    }
    if (active && p.final_state) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int j = 0; j < CT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * d + 4 * q4 + r, col = col0 + 16 * j + n;
                    if (row < p.dk && col < p.dv) p.final_state[sbase + (int64_t)row * p.dv + col] = S[d][j][r];
                }
    }
    // padding behind the sequence's end
    const int c0 = slice * NW * CT * 16, cn = (p.dv - c0) < NW * CT * 16 ? (p.dv - c0) : NW * CT * 16;
    for (int t = len + w; t < p.seqlen; t += NW)
        for (int cc = lane; cc < cn; cc += 64) ob[(int64_t)t * p.out_seq_stride + c0 + cc] = static_cast<T>(0.f);
}

// ---- host ----------------------------------------------------------------------------------------------------
int validate(const vms_gated_delta_params& p) {
    VMS_CHECK(p.dtype == VMS_F32 || p.dtype == VMS_F16 || p.dtype == VMS_BF16, "dtype must be fp32/fp16/bf16");
    VMS_CHECK(p.gate_dtype == VMS_F32 || p.gate_dtype == p.dtype, "g and beta must be fp32 or of the activations' type");
    VMS_CHECK(p.batch > 0 && p.seqlen > 0 && p.heads > 0 && p.heads_k > 0, "empty problem");
    VMS_CHECK(p.heads % p.heads_k == 0, "heads must be a multiple of heads_k");
    VMS_CHECK(p.dk >= 1 && p.dk <= 128, "key heads of 1 .. 128");
    VMS_CHECK(p.dv >= 1 && p.dv <= 4096, "value heads of 1 .. 4096");
    VMS_CHECK(p.heads <= 65535 && p.batch <= 65535 && p.seqlen <= (1 << 30), "problem too large");
    VMS_CHECK((int64_t)p.batch * p.heads * ((p.dv + 15) / 16) < (1LL << 31), "problem too large");
    VMS_CHECK(p.q && p.k && p.v && p.g && p.beta, "q, k, v, g, beta are required");
    const Layout l = layout(p);
    VMS_CHECK(p.workspace != nullptr && p.workspace_bytes >= l.bytes, "workspace is too small (vms_gated_delta_workspace_bytes)");
    VMS_CHECK((reinterpret_cast<uintptr_t>(p.workspace) & 15) == 0, "workspace must be 16-byte aligned");
    return VMS_OK;
}

template <typename T, int KP, int NW, int CT>
static int scan_launch(const vms_gated_delta_params& p, const Layout& l, hipStream_t s) {
    constexpr int NX = Prec<T>::NX, NS = Prec<T>::NS;
    constexpr int lds = 2 * NX * tile_bytes<KP>() + 2 * NS * kTri + 3 * C * 4;
    static_assert(NW * 64 >= 3 * C, "a thread per gate");
    static PerDeviceOnce once;
    if (lds > 65536) {
        const hipError_t e = once.run([&] {
            return hipFuncSetAttribute(reinterpret_cast<const void*>(&gd_scan_kernel<T, KP, NW, CT>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        });
        if (e != hipSuccess) { set_error("hipFuncSetAttribute: %s", hipGetErrorString(e)); return VMS_ERR_LAUNCH; }
    }
    const int slices = (l.vpad + NW * CT * 16 - 1) / (NW * CT * 16);
    hipLaunchKernelGGL((gd_scan_kernel<T, KP, NW, CT>), dim3(p.batch * p.heads * slices), dim3(NW * 64), lds, s, p, l, slices);
    VMS_LAUNCH_CHECK();
    return VMS_OK;
}
template <typename T, int KP>
static int fwd_launch(const vms_gated_delta_params& p, hipStream_t s) {
    const Layout l = layout(p);
    hipLaunchKernelGGL((gd_prep_kernel<T, KP>), dim3(l.chunks, p.heads, p.batch), dim3(64), 0, s, p, l);
    VMS_LAUNCH_CHECK();
    return scan_launch<T, KP, 4, 1>(p, l, s);
}
template <typename T>
static int fwd_type(const vms_gated_delta_params& p, hipStream_t s) {
    return pad_k(p.dk) == 64 ? fwd_launch<T, 64>(p, s) : fwd_launch<T, 128>(p, s);
}

}  // namespace gd
}  // namespace vms

using namespace vms;

extern "C" int64_t vms_gated_delta_workspace_bytes(const vms_gated_delta_params* pp) {
    if (!pp || pp->batch <= 0 || pp->seqlen <= 0 || pp->heads <= 0 || pp->dk <= 0 || pp->dv <= 0) return 0;
    return gd::layout(*pp).bytes;
}
extern "C" int64_t vms_gated_delta_bwd_workspace_bytes(const vms_gated_delta_params* pp) {
    if (!pp || pp->batch <= 0 || pp->seqlen <= 0 || pp->heads <= 0 || pp->dk <= 0 || pp->dv <= 0) return 0;
    return gd::layout(*pp).bwd_bytes;
}

extern "C" int vms_gated_delta_fwd(const vms_gated_delta_params* pp, void* stream) {
    VMS_CHECK(pp != nullptr, "null params");
    const vms_gated_delta_params& p = *pp;
    if (int rc = gd::validate(p)) return rc;
    VMS_CHECK(p.out != nullptr, "out is required");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int rc = p.dtype == VMS_BF16 ? gd::fwd_type<bf16_t>(p, s) : p.dtype == VMS_F16 ? gd::fwd_type<f16_t>(p, s) : gd::fwd_type<float>(p, s);
    if (rc == VMS_OK) set_last_kernel("gated_delta_fwd");
    return rc;
}
extern "C" int vms_sizeof_gated_delta_params(void) { return (int)sizeof(vms_gated_delta_params); }
