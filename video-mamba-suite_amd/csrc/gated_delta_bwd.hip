// gated_delta_bwd.hip -- gated delta rule, backward (vms_gated_delta_bwd); algebra, precision and layouts: gated_delta.h.
//
// With S0, U, T, M of every chunk from the forward's workspace and dS1 = the adjoint of a chunk's last state:
//   gd_bwd_scan  walks the chunks from the end, a workgroup per 16 CT columns of dS as in the forward:
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
#include <type_traits>

#include "gated_delta.h"

namespace vms {
namespace gd {

struct BwdArgs {   // what the kernels need of vms_gated_delta_bwd_params (one kernel argument block)
    vms_gated_delta_bwd_params q;
    Layout l;
};

// ---- the walk over the chunks, from the end ------------------------------------------------------------------
// Split among eight waves as the forward's walk: of the chain's four, wave w has token tile w of dU and Y and dk / 4 rows of dS; the other four load, make
// what depends on no dS (M^T dO, the planes of dO and of scale gam dO) and store.  Bound by the chain (K dS1 -> dU -> Y -> dS0): (8, 3136, 6 heads, 128 x 128) bf16
// 3.4 us per chunk, 169 us, 7200 cycles of which LDS works 3100, 1170 on bank conflicts; with one plane for what is stored 131 us, all of it on four waves then 164 us.
template <typename T, int NB, int KP, int CT, int FIT>
struct BwdScanLds {   // bytes and places in LDS
    static constexpr int NX = Prec<T>::NX;
    static constexpr int kK = NX * tile_bytes<KP>(), kPiece = VTile<T, CT, FIT != 0>::kBytes, kSum = 4 * CT * 1024;
    static constexpr int S = 0, O = S + Exchange<NB, CT, KP>::kBytes, G = O + Exchange<NX, CT, C>::kBytes, U = G + Exchange<NB, CT, C>::kBytes,
                         Y = U + Exchange<NB, CT, C>::kBytes, E = Y + Exchange<NB, CT, C>::kBytes, V = E + kSum, B = V + 4 * kPiece, K = B + 2 * 4 * GateTile::kBytes;
    static constexpr bool kStaged = K + 4 * kK <= 163840;   // two tiles each of K and Q; else one each, and K straight into the chain's registers
    static constexpr int Q = K + (kStaged ? 2 : 1) * kK, kBytes = Q + (kStaged ? 2 : 1) * kK;
};

template <typename T, int NB, int KP, int CT, int FIT>
__global__ __launch_bounds__(512, 1) void gd_bwd_scan_kernel(const BwdArgs a, const int slices) {
    constexpr int NX = Prec<T>::NX, kT = NS + Prec<T>::NO, kM = kT + NB;   // planes of a chunk's slot before the transposes of T, of M
    constexpr int KB = KP / 32, DW = KP / 64;
    constexpr bool WHOLE = FIT != 0;
    using Lds = BwdScanLds<T, NB, KP, CT, FIT>;
    static_assert(Lds::kBytes <= 163840, "160 KB of LDS");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const Exchange<NB, CT, KP> Sx{lds + Lds::S};
    const Exchange<NX, CT, C> Ox{lds + Lds::O};                                        // dO
    const Exchange<NB, CT, C> Gx{lds + Lds::G}, Ux{lds + Lds::U}, Yx{lds + Lds::Y};   // scale gam dO, dU, -beta gam Y

    const vms_gated_delta_params& p = a.q.f;
    const Layout& l = a.l;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, q4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), w = wave & 3;
    int pair, slice;
    pair_of(blockIdx.x, p.batch * p.heads, slices, pair, slice);
    const int b = pair / p.heads, h = pair % p.heads, hk = h / (p.heads / p.heads_k);
    const int len = length_of(p, b), nc = (len + C - 1) / C;
    const int col0 = slice * CT * 16;
    const Rows<T> K(p.k, (int64_t)b * p.k_batch_stride + (int64_t)hk * p.k_head_stride, p.k_seq_stride, len, p.reverse);
    const char* const ws = static_cast<const char*>(p.workspace);
    char* const wb = static_cast<char*>(a.q.workspace);
    const int64_t slot0 = (int64_t)pair * l.chunks;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    auto k_tile = [&](int odd) __attribute__((always_inline)) { return lds + Lds::K + (Lds::kStaged ? odd * Lds::kK : 0); };
    auto q_tile = [&](int odd) __attribute__((always_inline)) { return lds + Lds::Q + (Lds::kStaged ? odd * Lds::kK : 0); };
    auto g_at = [&](int odd) __attribute__((always_inline)) { return GateTile{reinterpret_cast<float*>(lds + Lds::B + (4 * odd + w) * GateTile::kBytes), 0.f}; };
    f32x4* const sums = reinterpret_cast<f32x4*>(lds + Lds::E) + 64 * CT * w + lane;   // M^T dO to the chain, Y from it: fp32, lane by lane
    auto fetch_rows = [&](const Rows<T>& x, int c, Raw8<T> (&r)[KB]) __attribute__((always_inline)) {   // operands: token 16 w + n
        const int at = c * C + 16 * w + n;
        const T* const row = x.row(at < len ? at : len - 1);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) r[kb] = fit_load<FIT, T>(row, 32 * kb + 8 * q4, p.dk);
    };
    auto piece_row = [&](int i) __attribute__((always_inline)) { return (lane + 64 * i) / (KP / 8); };   // the same 16 rows by lines: piece i of 8 columns
    auto piece_col = [&](int i) __attribute__((always_inline)) { return 8 * ((lane + 64 * i) % (KP / 8)); };
    auto fetch_lines = [&](const Rows<T>& x, int c, Raw8<T> (&r)[KB]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KB; ++i) {
            const int at = c * C + 16 * w + piece_row(i);
            r[i] = fit_load<FIT, T>(x.row(at < len ? at : len - 1), piece_col(i), p.dk);
        }
    };
    auto fetch_tri = [&](int c, int first, Frag<NB> (&f)[2]) __attribute__((always_inline)) {   // columns 16 w + n (row blocks 0, 1; tiles 2 and 3 have no block 0)
        const char* const at = ws + l.tri + (slot0 + c) * l.tri_slot + first * kTri;            // first: kT, kM
        f[0] = tri_cols<NB>(at, w, w >= 2 ? 1 : 0, lane);
        f[1] = tri_cols<NB>(at, w, 1, lane);
    };
    auto before = [&](int c, int by) __attribute__((always_inline)) { return c > by ? c - by : 0; };
    // Both sides below meet at three barriers per chunk: dS and M^T dO are there; dU is there; Y is there
    if (wave < 4) {
        // ---- the chain: dU, Y, dS
        __builtin_amdgcn_s_setprio(2);   // the other wave of this SIMD has slack
        f32x4 dS[DW][CT];
        const int64_t sbase = (int64_t)pair * p.dk * p.dv;
#pragma unroll
        for (int d = 0; d < DW; ++d)
#pragma unroll
            for (int j = 0; j < CT; ++j) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * (DW * w + d) + 4 * q4 + r, col = col0 + col_of<CT>(j, n);
                    dS[d][j][r] = a.q.dfinal_state && row < p.dk && col < p.dv ? a.q.dfinal_state[sbase + (int64_t)row * p.dv + col] : 0.f;
                }
                Sx.put(j, n, 16 * (DW * w + d) + 4 * q4, dS[d][j]);
            }
        Raw8<T> kr[KB];
        auto chunk = [&](int c, auto odd_c, Frag<NB> (&tf)[2]) __attribute__((always_inline)) {
            constexpr int odd = decltype(odd_c)::value;
            char* const Ks = k_tile(odd);
            const char* const Qs = q_tile(odd);
            const GateTile gt = g_at(odd);
            __syncthreads();   // (not staged) K's tile is no longer read
            // dU = del K dS1 + M^T dO
            f32x4 dU[CT];
#pragma unroll
            for (int j = 0; j < CT; ++j) dU[j] = zero;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                Frag<NX> kf;
                if constexpr (Lds::kStaged) {
                    kf = tile_rows<KP, NX>(Ks, 16 * w + n, 32 * kb + 8 * q4);
                } else {
                    kf = planes_of<T>(fit_clear<FIT, T>(kr[kb], 32 * kb + 8 * q4, p.dk));
                    tile_put<KP, NX>(Ks, 16 * w + n, 32 * kb + 8 * q4, kf);
                }
#pragma unroll
                for (int j = 0; j < CT; ++j) mma<NB>(dU[j], kf, Sx.get(j, n, 32 * kb + 8 * q4));
            }
            if constexpr (!Lds::kStaged) fetch_rows(K, before(c, 1), kr);
            const f32x4 ga = gt.four(0, q4), be = gt.four(1, q4), de = gt.four(2, q4);
            const float glast = gt.last();
#pragma unroll
            for (int j = 0; j < CT; ++j) Ux.put(j, n, paired(w, q4), dU[j] * de + sums[64 * j]);
            __syncthreads();
            // Y = T^T dU
            f32x4 Y[CT];
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                Y[j] = zero;
                mma<NB>(Y[j], tf[1], Ux.get(j, n, 32 + 8 * q4));
            }
            if (w < 2) {
#pragma unroll
                for (int j = 0; j < CT; ++j) mma<NB>(Y[j], tf[0], Ux.get(j, n, 8 * q4));
                settle(Y);
            }
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                sums[64 * j] = Y[j];
                f32x4 x;
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = -ga[r] * (be[r] * Y[j][r]);
                Yx.put(j, n, paired(w, q4), x);
            }
            __syncthreads();
            // dS0 = gam dS1 + Q^T (scale gam dO) - K^T (beta gam Y)
#pragma unroll
            for (int d = 0; d < DW; ++d)
#pragma unroll
                for (int j = 0; j < CT; ++j) dS[d][j] *= glast;
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                Frag<NB> gf[CT], yf[CT];
#pragma unroll
                for (int j = 0; j < CT; ++j) { gf[j] = Gx.get(j, n, 32 * tb + 8 * q4); yf[j] = Yx.get(j, n, 32 * tb + 8 * q4); }
#pragma unroll
                for (int d = 0; d < DW; ++d) {
                    const Frag<NX> qc = tile_cols<KP, NX>(Qs, DW * w + d, tb, n, q4), kc = tile_cols<KP, NX>(Ks, DW * w + d, tb, n, q4);
#pragma unroll
                    for (int j = 0; j < CT; ++j) {
                        mma<NB>(dS[d][j], qc, gf[j]);
                        mma<NB>(dS[d][j], kc, yf[j]);
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < DW; ++d)
#pragma unroll
                for (int j = 0; j < CT; ++j) Sx.put(j, n, 16 * (DW * w + d) + 4 * q4, dS[d][j]);
            fetch_tri(before(c, 2), kT, tf);
        };
        if (nc > 0) {
            Frag<NB> t0[2], t1[2];
            if constexpr (!Lds::kStaged) fetch_rows(K, nc - 1, kr);
            fetch_tri(nc - 1, kT, t0);
            fetch_tri(before(nc - 1, 1), kT, t1);
            __syncthreads();   // dO of the last chunk is there, for the other side
            for (int c = nc - 1;;) {
                chunk(c, std::integral_constant<int, 0>{}, t0);
                if (--c < 0) break;
                chunk(c, std::integral_constant<int, 1>{}, t1);
                if (--c < 0) break;
            }
        }
        if (a.q.dinitial_state) {
#pragma unroll
            for (int d = 0; d < DW; ++d)
#pragma unroll
                for (int j = 0; j < CT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = 16 * (DW * w + d) + 4 * q4 + r, col = col0 + col_of<CT>(j, n);
                        if (row < p.dk && col < p.dv) a.q.dinitial_state[sbase + (int64_t)row * p.dv + col] = dS[d][j][r];
                    }
        }
    } else {
        // ---- what both sides read, dS and Y for the gradients, dV
        const Rows<T> Q(p.q, (int64_t)b * p.q_batch_stride + (int64_t)hk * p.q_head_stride, p.q_seq_stride, len, p.reverse);
        const Rows<T> dO(a.q.dout, (int64_t)b * a.q.dout_batch_stride + (int64_t)h * a.q.dout_head_stride, a.q.dout_seq_stride, len, p.reverse);
        const int64_t dv_seq = (int64_t)p.heads * p.dv;
        const Rows<T> dV(a.q.dv, ((int64_t)b * p.seqlen * p.heads + h) * p.dv, dv_seq, len, p.reverse);
        struct Ahead {
            Raw8<T> k[KB], q[KB];
            VTile<T, CT, WHOLE> o;   // dO
            GateTile g;
        };
        const OTile<T, CT, WHOLE> ot{lds + Lds::V + w * Lds::kPiece};   // (dO's place: handed on before dV comes, stored before the next dO)
        auto fetch_k = [&](int c, Ahead& x) __attribute__((always_inline)) {
            if constexpr (Lds::kStaged) fetch_lines(K, c, x.k);
        };
        auto fetch_q = [&](int c, Ahead& x) __attribute__((always_inline)) {
            if constexpr (Lds::kStaged) fetch_lines(Q, c, x.q);
        };
        auto fetch_small = [&](int c, Ahead& x) __attribute__((always_inline)) {
            x.o.fetch(dO, c * C + 16 * w, len, col0, p.dv, lane);
            x.g.fetch(reinterpret_cast<const float*>(reinterpret_cast<const Gates*>(ws + l.gates) + slot0 + c), w, lane);
        };
        f32x4 scaled[CT];   // of the chunk that was handed over last: the place of the one before is read until the barrier
        auto hand = [&](int c, auto odd_c, Ahead& x) __attribute__((always_inline)) {   // into LDS
            constexpr int odd = decltype(odd_c)::value;
            if constexpr (Lds::kStaged) {
#pragma unroll
                for (int i = 0; i < KB; ++i) {
                    tile_put<KP, NX>(k_tile(odd), 16 * w + piece_row(i), piece_col(i), planes_of<T>(fit_clear<FIT, T>(x.k[i], piece_col(i), p.dk)));
                    tile_put<KP, NX>(q_tile(odd), 16 * w + piece_row(i), piece_col(i), planes_of<T>(fit_clear<FIT, T>(x.q[i], piece_col(i), p.dk)));
                }
            }
            x.o.base = lds + Lds::V + w * Lds::kPiece;
            x.g.base = g_at(odd).base;
            x.o.hand(c * C + 16 * w, len, col0, p.dv, lane, false);
            x.g.hand(lane);
            const f32x4 ga = x.g.four(0, q4);
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                const f32x4 g = x.o.get(j, n, q4);
                Ox.put(j, n, paired(w, q4), g);
#pragma unroll
                for (int r = 0; r < 4; ++r) scaled[j][r] = p.scale * ga[r] * g[r];
            }
        };
        auto other_grad = [&](const Frag<NB> (&mf)[2]) __attribute__((always_inline)) {   // M^T dO
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                f32x4 e = zero;
                mma<NB>(e, mf[1], Ox.get(j, n, 32 + 8 * q4));
                if (w < 2) {
                    mma<NB>(e, mf[0], Ox.get(j, n, 8 * q4));
                    settle(e);
                }
                sums[64 * j] = e;
            }
        };
        Raw8<T> qr[KB];
        auto chunk = [&](int c, auto odd_c, Ahead& mine, Ahead& other, Frag<NB> (&mf)[2]) __attribute__((always_inline)) {   // other, mf: of chunk c - 1
            constexpr int odd = decltype(odd_c)::value;
            const int64_t slot = slot0 + c;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < CT; ++j) Gx.put(j, n, paired(w, q4), scaled[j]);
            if (c + 1 < nc) ot.store(dV, (c + 1) * C + 16 * w, len, col0, p.dv, lane);
            if constexpr (!Lds::kStaged) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) tile_put<KP, NX>(q_tile(0), 16 * w + n, 32 * kb + 8 * q4, planes_of<T>(fit_clear<FIT, T>(qr[kb], 32 * kb + 8 * q4, p.dk)));
                fetch_rows(Q, before(c, 1), qr);
            }
            if (w < KB) {
                Frag<NB> sf[CT];
#pragma unroll
                for (int j = 0; j < CT; ++j) sf[j] = Sx.get(j, n, 32 * w + 8 * q4);
                store_frag<NB, CT, false>(wb + l.dS + slot * l.s_slot, KP, l.vpad, 32 * w, 0, col0, sf, n, q4);
            }
            fetch_k(before(c, 2), mine);
            __syncthreads();
            hand(before(c, 1), std::integral_constant<int, 1 - odd>{}, other);
            fetch_small(before(c, 3), other);
            __syncthreads();
            fetch_q(before(c, 3), other);
            f32x4 Y[CT], dv[CT];
            const f32x4 be = g_at(odd).four(1, q4);
#pragma unroll
            for (int j = 0; j < CT; ++j) Y[j] = sums[64 * j];
            other_grad(mf);
            fetch_tri(before(c, 3), kM, mf);
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                const Frag<NB> f = frag_of<NB>(be * Y[j], zero);
                dv[j] = zero;
#pragma unroll
                for (int i = NB - 1; i >= 0; --i) dv[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.p[i], unit_frag(0, n, q4), dv[j], 0, 0, 0);
            }
            store_rows<NB, CT>(wb + l.Y + slot * l.u_slot, C, l.vpad, 16 * w, col0, Y, n, q4);
            ot.put(dv, lane);
        };
        if (nc > 0) {
            Ahead a0, a1;
            Frag<NB> m0[2], m1[2];
            if constexpr (!Lds::kStaged) fetch_rows(Q, nc - 1, qr);
            auto fetch = [&](int c, Ahead& x) __attribute__((always_inline)) { fetch_k(c, x); fetch_q(c, x); fetch_small(c, x); };
            fetch(nc - 1, a0);
            fetch(before(nc - 1, 1), a1);
            fetch_tri(nc - 1, kM, m0);
            fetch_tri(before(nc - 1, 1), kM, m1);
            hand(nc - 1, std::integral_constant<int, 0>{}, a0);
            fetch_q(before(nc - 1, 2), a0);
            fetch_small(before(nc - 1, 2), a0);
            __syncthreads();
            other_grad(m0);
            fetch_tri(before(nc - 1, 2), kM, m0);
            for (int c = nc - 1;;) {
                chunk(c, std::integral_constant<int, 0>{}, a0, a1, m1);
                if (--c < 0) break;
                chunk(c, std::integral_constant<int, 1>{}, a1, a0, m0);
                if (--c < 0) break;
            }
            ot.store(dV, 16 * w, len, col0, p.dv, lane);
        }
        T* const dvb = static_cast<T*>(a.q.dv) + ((int64_t)b * p.seqlen * p.heads + h) * p.dv;   // padding behind the sequence's end
        const int cn = p.dv - col0 < CT * 16 ? p.dv - col0 : CT * 16;
        for (int t = len + w; t < p.seqlen; t += 4)
            for (int cc = lane; cc < cn; cc += 64) dvb[(int64_t)t * dv_seq + col0 + cc] = static_cast<T>(0.f);
    }
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

// Stage 1 walks v 32 columns at a time: U, Y, dO (64 rows) and S0, dS1 (KP rows) go through registers (the next block is on its way while this one is
// multiplied) into LDS, 16-byte operands from there; the sums that need no product (Y.V, <S0, dS1>) are taken from the pieces as they pass.  Eight waves:
// wave w has token tile w % 4 of dQ and W (w < 4: "left", what depends on the token as the later one) or of X (w >= 4: "right"), so that no product is
// made twice and the accumulators fit.  (8, 3136, 6 heads, 128 x 128) bf16: 278 us for 0.69 GB and 70 GFLOP of bf16 products (145 us for
// 0.45 GB and 36 GFLOP with one plane); bound by the steps between the barriers (a workgroup of eight waves fills a CU's registers) and by LDS, half of whose cycles
// are bank conflicts.  Stage 2 multiplies the 64 x 64 results with Q and K, whose tiles take stage 1's place in LDS.
template <typename T, int NB, int KP, bool WHOLE, bool SHARED>   // WHOLE: dk % 8 == 0 and dv % 8 == 0; SHARED: several heads per q / k head
__global__ __launch_bounds__(512, 2) void gd_grad_kernel(const BwdArgs a) {
    constexpr int NX = Prec<T>::NX, DT = KP / 16, TB = tile_bytes<KP>();
    constexpr int PK = C * KP / 8 / 512;   // 8-element pieces of a q / k tile per thread
    constexpr int ROW = 80;                 // bytes of 32 columns in LDS: 16 rows fall on all banks
    extern __shared__ __attribute__((aligned(16))) char lds[];
    Gates* const gs = reinterpret_cast<Gates*>(lds);
    float* const dGs = reinterpret_cast<float*>(gs + 1);
    float* const kxs = dGs + C;
    float* const yvs = kxs + C;
    float* const part = yvs + C;   // one sum per wave
    char* const big = reinterpret_cast<char*>(part + 8);
    char* const Ks = big;          // stage 2
    char* const Qs = Ks + NX * TB;
    f32x4* const Wx = reinterpret_cast<f32x4*>(Qs + NX * TB);   // beta W, from the left wave to the right one
    char* const Us = big;          // stage 1
    char* const Ys = Us + NB * C * ROW;
    char* const Os = Ys + NB * C * ROW;
    char* const Ss = Os + NX * C * ROW;
    char* const Ds = Ss + NB * KP * ROW;

    const vms_gated_delta_params& p = a.q.f;
    const Layout& l = a.l;
    const int tid = threadIdx.x, lane = tid & 63, w8 = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, q4 = lane >> 4;
    const int w = w8 & 3;
    const bool left = w8 < 4;
    const int c = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
    const int rep = SHARED ? p.heads / p.heads_k : 1;
    const int len = length_of(p, b);
    const int64_t dk_seq = (int64_t)p.heads_k * p.dk;
    T* const dqb = static_cast<T*>(a.q.dq) + ((int64_t)b * p.seqlen * p.heads_k + hk) * p.dk;
    T* const dkb = static_cast<T*>(a.q.dk) + ((int64_t)b * p.seqlen * p.heads_k + hk) * p.dk;

    // padding rows of this chunk
    {
        const int first = c * C > len ? c * C : len, end = (c + 1) * C < p.seqlen ? (c + 1) * C : p.seqlen;
        for (int t = first + w8; t < end; t += 8) {
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

    const Rows<T> Q(p.q, (int64_t)b * p.q_batch_stride + (int64_t)hk * p.q_head_stride, p.q_seq_stride, len, p.reverse);
    const Rows<T> K(p.k, (int64_t)b * p.k_batch_stride + (int64_t)hk * p.k_head_stride, p.k_seq_stride, len, p.reverse);
    const char* const ws = static_cast<const char*>(p.workspace);
    const char* const wb = static_cast<const char*>(a.q.workspace);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const int own = 16 * w + n, at_own = c * C + own;   // this lane's token
    const bool ok_own = at_own < len;
    // stage 1: a thread's piece of U and dO (left) or Y and V (right), of S0 and dS1
    const int prow = (tid & 255) >> 2, pcol = 8 * (tid & 3), srow = (tid >> 2) & (KP - 1);
    const bool has_s = tid < 4 * KP;
    const int at_p = c * C + prow;
    const bool ok_p = at_p < len;
    // dQ (left), dK (right): a wave's 16 rows through its own part of Q's or K's tile, which nobody reads any more, to whole lines (8-byte pieces of 16 rows at
    // once cost the memory pipe 64 accesses a store instead of 16)
    auto store_grad = [&](const f32x4 (&x)[DT]) __attribute__((always_inline)) {
        constexpr int PITCH = KP * (int)sizeof(T) + 16;
        static_assert(C * PITCH <= NX * TB, "a tile's place");
        char* const mine = (left ? Qs : Ks) + 16 * w * PITCH;
        T* const base = left ? dqb : dkb;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const T o[4] = {static_cast<T>(x[d][0]), static_cast<T>(x[d][1]), static_cast<T>(x[d][2]), static_cast<T>(x[d][3])};
            __builtin_memcpy(__builtin_assume_aligned(mine + n * PITCH + (16 * d + 4 * q4) * (int)sizeof(T), 8), o, sizeof(o));
        }
#pragma unroll
        for (int i = 0; i < KP / 32; ++i) {
            const int id = lane + 64 * i, row = id / (KP / 8), cc = 8 * (id % (KP / 8)), at = c * C + 16 * w + row;
            Raw8<T> r;
            __builtin_memcpy(&r, __builtin_assume_aligned(mine + row * PITCH + cc * (int)sizeof(T), 16), sizeof(r));
            if (at < len) {
                T* const to = base + token(at, len, p.reverse) * dk_seq + cc;
                if (WHOLE) {
                    if (cc < p.dk) __builtin_memcpy(to, &r, sizeof(r));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (cc + e < p.dk) to[e] = r.v[e];
                }
            }
        }
    };
    f32x4 total[SHARED ? DT : 1];   // dQ (left), dK (right) over the heads
    if constexpr (SHARED)
#pragma unroll
        for (int d = 0; d < DT; ++d) total[d] = zero;

    for (int r = 0; r < rep; ++r) {
        const int h = hk * rep + r;
        const int64_t slot = ((int64_t)b * p.heads + h) * l.chunks + c;
        const char* const Aw = left ? ws + l.U + slot * l.u_slot : wb + l.Y + slot * l.u_slot;
        const char* const Sw = ws + l.S0 + slot * l.s_slot;
        const char* const Dw = wb + l.dS + slot * l.s_slot;
        const Rows<T> V(p.v, (int64_t)b * p.v_batch_stride + (int64_t)h * p.v_head_stride, p.v_seq_stride, len, p.reverse);
        const Rows<T> dO(a.q.dout, (int64_t)b * a.q.dout_batch_stride + (int64_t)h * a.q.dout_head_stride, a.q.dout_seq_stride, len, p.reverse);
        const T* const brow = (left ? dO : V).row(ok_p ? at_p : len - 1);
        Frag<NB> ap, sp, dp;
        Raw8<T> bp;
        auto fetch = [&](int vk) __attribute__((always_inline)) {
            const int cc = 32 * vk + pcol;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                ap.p[i] = *reinterpret_cast<const bf16x8*>(Aw + 2 * (((int64_t)i * C + prow) * l.vpad + cc));
                sp.p[i] = *reinterpret_cast<const bf16x8*>(Sw + 2 * (((int64_t)i * KP + srow) * l.vpad + cc));
                dp.p[i] = *reinterpret_cast<const bf16x8*>(Dw + 2 * (((int64_t)i * KP + srow) * l.vpad + cc));
            }
            bp = load_raw8<WHOLE, T>(brow, cc, p.dv);
        };
        float yv = 0.f, ss = 0.f;   // this thread's part of Y.V (its token), of <S0, dS1>
        auto value = [&](const Frag<NB>& f, int e) __attribute__((always_inline)) {
            float x = 0.f;
#pragma unroll
            for (int i = NB - 1; i >= 0; --i) x += static_cast<float>(f.p[i][e]);
            return x;
        };
        auto hand = [&](int vk) __attribute__((always_inline)) {
            const int cc = 32 * vk + pcol;
            const Raw8<T> b8 = clear<WHOLE, T>(bp, cc, p.dv, ok_p);
            char* const at = (left ? Us : Ys) + prow * ROW + 2 * pcol;
            char* const as = Ss + srow * ROW + 2 * pcol;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                *reinterpret_cast<bf16x8*>(at + i * C * ROW) = ap.p[i];
                if (has_s) {
                    *reinterpret_cast<bf16x8*>(as + i * KP * ROW) = sp.p[i];
                    *reinterpret_cast<bf16x8*>(as + (Ds - Ss) + i * KP * ROW) = dp.p[i];
                }
            }
            if (has_s)
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(value(sp, e), value(dp, e), ss);
            if (left) {
                const Frag<NX> of = planes_of<T>(b8);
#pragma unroll
                for (int i = 0; i < NX; ++i) *reinterpret_cast<bf16x8*>(Os + (i * C + prow) * ROW + 2 * pcol) = of.p[i];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) yv = fmaf(value(ap, e), static_cast<float>(b8.v[e]), yv);
            }
        };
        auto from = [&](const char* base, int rows, int row, auto planes) __attribute__((always_inline)) {
            Frag<decltype(planes)::value> f;
#pragma unroll
            for (int i = 0; i < decltype(planes)::value; ++i) f.p[i] = *reinterpret_cast<const bf16x8*>(base + (i * rows + row) * ROW + 16 * q4);
            return f;
        };
        constexpr std::integral_constant<int, NB> nb{};
        constexpr std::integral_constant<int, NX> nx{};
        // 64 x 64 products [j][i]: rows = another tile's tokens, columns (lanes) = this wave's.  left: m = dO_i.U_j, z = Y_i.U_j with this wave's tokens as i
        // (tiles j <= w); right: with this wave's tokens as j (tiles i >= w).  A: left dO S0^T -> dQ, right U dS1^T -> X;  B: left Y S0^T -> W
        f32x4 m[4], z[4], A[DT], B[DT];
#pragma unroll
        for (int t = 0; t < 4; ++t) { m[t] = zero; z[t] = zero; }
#pragma unroll
        for (int d = 0; d < DT; ++d) { A[d] = zero; B[d] = zero; }
        auto multiply = [&]() __attribute__((always_inline)) {
            if (left) {
                const Frag<NB> yi = from(Ys, C, own, nb);
                const Frag<NX> oi = from(Os, C, own, nx);
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    if (t <= w) {
                        const Frag<NB> uj = from(Us, C, 16 * t + n, nb);
                        mma<NB>(m[t], uj, oi);
                        mma<NB>(z[t], uj, yi);
                        asm volatile("" : "+v"(m[t]));
                        settle(z[t]);
                    }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const Frag<NB> s0 = from(Ss, KP, 16 * d + n, nb);
                    mma<NB>(A[d], s0, oi);
                    mma<NB>(B[d], s0, yi);
                }
                settle(A, B);
            } else {
                const Frag<NB> ui = from(Us, C, own, nb);
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    if (t >= w) {
                        mma<NB>(m[t], from(Os, C, 16 * t + n, nx), ui);
                        mma<NB>(z[t], from(Ys, C, 16 * t + n, nb), ui);
                        asm volatile("" : "+v"(m[t]));
                        settle(z[t]);
                    }
#pragma unroll
                for (int d = 0; d < DT; ++d) mma<NB>(A[d], from(Ds, KP, 16 * d + n, nb), ui);
                settle(A);
            }
        };
        const int blocks = l.vpad / 32;
        fetch(0);
        for (int vk = 0; vk < blocks; ++vk) {
            __syncthreads();   // LDS is free
            hand(vk);
            fetch(vk + 1 < blocks ? vk + 1 : vk);
            __syncthreads();
            multiply();
        }
        Raw8<T> kr[PK], qr[PK];
#pragma unroll
        for (int i = 0; i < PK; ++i) {
            const int id = tid + i * 512, row = id / (KP / 8), cc = 8 * (id % (KP / 8)), at = c * C + row;
            kr[i] = load_raw8<WHOLE, T>(K.row(at < len ? at : len - 1), cc, p.dk);
            qr[i] = load_raw8<WHOLE, T>(Q.row(at < len ? at : len - 1), cc, p.dk);
        }
        if (tid < (int)(sizeof(Gates) / 4))
            reinterpret_cast<float*>(gs)[tid] = reinterpret_cast<const float*>(reinterpret_cast<const Gates*>(ws + l.gates) + slot)[tid];
        yv += __shfl_xor(yv, 1);
        yv += __shfl_xor(yv, 2);
        if (!left && (tid & 3) == 0) yvs[prow] = yv;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PK; ++i) {
            const int id = tid + i * 512, row = id / (KP / 8), cc = 8 * (id % (KP / 8));
            const bool ok = c * C + row < len;
            tile_put<KP, NX>(Ks, row, cc, planes_of<T>(clear<WHOLE, T>(kr[i], cc, p.dk, ok)));
            tile_put<KP, NX>(Qs, row, cc, planes_of<T>(clear<WHOLE, T>(qr[i], cc, p.dk, ok)));
        }
        __syncthreads();
        const double Gi = gs->G[own];
        auto rowdot = [&](const char* tile, const f32x4 (&x)[DT]) __attribute__((always_inline)) {
            float s = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                f32x4 v = zero;
#pragma unroll
                for (int i = NX - 1; i >= 0; --i) {
                    const bf16x4 t4 = *reinterpret_cast<const bf16x4*>(tile + i * TB + own * tile_row<KP>() + 2 * (16 * d + 4 * q4));
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += static_cast<float>(t4[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s = fmaf(v[e], x[d][e], s);
            }
            return s;
        };
        // the 64 x 64 factors in the state's precision: dg is a difference of sums over pairs, which cancel only as far as the two
        // roundings of a pair agree
        if (left) {
            const float gi = gs->gam[own], bi = gs->bet[own];
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    A[d][e] *= p.scale * gi;
                    B[d][e] *= gi;
                }
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (t <= w) {
                    const f64x4 Gj = *reinterpret_cast<const f64x4*>(&gs->G[16 * t + 4 * q4]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = 16 * t + 4 * q4 + e;
                        const float L = decay(j <= own, Gi - Gj[e]), x = L * z[t][e];
                        m[t][e] *= p.scale * L;
                        z[t][e] = j < own ? x : 0.f;
                    }
                }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
                if (2 * kb <= w) {
                    const Frag<NB> fm = frag_of<NB>(m[2 * kb], m[2 * kb + 1]), fz = frag_of<NB>(z[2 * kb], z[2 * kb + 1]);
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const Frag<NX> kc = tile_cols<KP, NX>(Ks, d, kb, n, q4);
                        mma<NB>(A[d], kc, fm);
                        mma<NB>(B[d], kc, fz);
                    }
                    settle(A, B);
                }
            const float qd = quarters_sum(rowdot(Qs, A)), kw = quarters_sum(rowdot(Ks, B));
#pragma unroll
            for (int d = 0; d < DT; ++d) Wx[(w * DT + d) * 64 + lane] = B[d] * bi;
            if (q4 == 0) {
                dGs[own] = qd - bi * kw;
                if (ok_own) st_gate(a.q.dbeta, ((int64_t)b * p.seqlen + token(at_own, len, p.reverse)) * p.heads + h, p.gate_dtype, yvs[own] - kw);
            }
        } else {
            const float di = gs->del[own];
#pragma unroll
            for (int d = 0; d < DT; ++d) A[d] *= di;
            ss = fmaf(gs->gam[C - 1], ss, rowdot(Ks, A));   // + the state's own part, below
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (t >= w) {
                    const f64x4 G4 = *reinterpret_cast<const f64x4*>(&gs->G[16 * t + 4 * q4]);
                    const f32x4 b4 = *reinterpret_cast<const f32x4*>(&gs->bet[16 * t + 4 * q4]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 16 * t + 4 * q4 + e;
                        const float L = decay(i >= own, G4[e] - Gi), x = -b4[e] * L * z[t][e];
                        m[t][e] *= p.scale * L;
                        z[t][e] = i > own ? x : 0.f;
                    }
                }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
                if (2 * kb + 1 >= w) {
                    const Frag<NB> fm = frag_of<NB>(m[2 * kb], m[2 * kb + 1]), fz = frag_of<NB>(z[2 * kb], z[2 * kb + 1]);
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        mma<NB>(A[d], tile_cols<KP, NX>(Qs, d, kb, n, q4), fm);
                        mma<NB>(A[d], tile_cols<KP, NX>(Ks, d, kb, n, q4), fz);
                    }
                    settle(A);
                }
            const float kx = quarters_sum(rowdot(Ks, A));
            if (q4 == 0) kxs[own] = kx;
        }
        ss = wave_sum(left ? gs->gam[C - 1] * ss : ss);
        if (lane == 0) part[w8] = ss;
        __syncthreads();
        if (w8 == 0) {   // lane = token
            float x = dGs[lane] - kxs[lane];
#pragma unroll
            for (int s = 1; s < 64; s *= 2) {
                const float o = __shfl_down(x, s);
                if (lane + s < 64) x += o;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) x += part[i];
            const int at = c * C + lane;
            if (at == 0 && !p.initial_state && !a.q.dinitial_state) x = 0.f;   // there is nothing that the first gate could forget: exact, where two equal terms would leave their roundings
            if (at < len) st_gate(a.q.dg, ((int64_t)b * p.seqlen + token(at, len, p.reverse)) * p.heads + h, p.gate_dtype, x);
        }
        if (!left)
#pragma unroll
            for (int d = 0; d < DT; ++d) A[d] -= Wx[(w * DT + d) * 64 + lane];   // dK
        if constexpr (SHARED) {
#pragma unroll
            for (int d = 0; d < DT; ++d) total[d] += A[d];
        } else {
            store_grad(A);
        }
    }
    if constexpr (SHARED) store_grad(total);
}

// ---- host ----------------------------------------------------------------------------------------------------
template <typename T, int NB, int KP, int CT, int FIT>
static int bwd_scan_launch(const BwdArgs& a, hipStream_t s) {
    constexpr int lds = BwdScanLds<T, NB, KP, CT, FIT>::kBytes;
    static PerDeviceOnce once;
    if (int rc = allow_lds(once, reinterpret_cast<const void*>(&gd_bwd_scan_kernel<T, NB, KP, CT, FIT>), lds)) return rc;
    const int slices = (a.l.vpad + CT * 16 - 1) / (CT * 16);
    hipLaunchKernelGGL((gd_bwd_scan_kernel<T, NB, KP, CT, FIT>), dim3(a.q.f.batch * a.q.f.heads * slices), dim3(512), lds, s, a, slices);
    VMS_LAUNCH_CHECK();
    return VMS_OK;
}
template <typename T, int NB, int KP, int CT>
static int bwd_scan_fit(const BwdArgs& a, int fit, hipStream_t s) {
    return fit == 2 ? bwd_scan_launch<T, NB, KP, CT, 2>(a, s) : fit == 1 ? bwd_scan_launch<T, NB, KP, CT, 1>(a, s) : bwd_scan_launch<T, NB, KP, CT, 0>(a, s);
}
template <typename T, int NB, int KP, bool WHOLE, bool SHARED>
static int grad_launch(const BwdArgs& a, hipStream_t s) {
    constexpr int NX = Prec<T>::NX;
    constexpr int one = (2 * NB + NX) * C * 80 + 2 * NB * KP * 80, two = 2 * NX * tile_bytes<KP>() + C * KP * 4;
    constexpr int lds = (int)sizeof(Gates) + (3 * C + 8) * 4 + (one > two ? one : two);
    static_assert(lds <= 163840, "160 KB of LDS");
    static PerDeviceOnce once;
    if (int rc = allow_lds(once, reinterpret_cast<const void*>(&gd_grad_kernel<T, NB, KP, WHOLE, SHARED>), lds)) return rc;
    hipLaunchKernelGGL((gd_grad_kernel<T, NB, KP, WHOLE, SHARED>), dim3(a.l.chunks, a.q.f.heads_k, a.q.f.batch), dim3(512), lds, s, a);
    VMS_LAUNCH_CHECK();
    return VMS_OK;
}
template <typename T, int NB, int KP>
static int bwd_launch(const BwdArgs& a, hipStream_t s) {
    const int fit = fit_of(a.q.f.dk, a.q.f.dv);
    int rc;
    if constexpr (bwd_columns(sizeof(T) == 4 ? VMS_F32 : std::is_same_v<T, f16_t> ? VMS_F16 : VMS_BF16, NB, KP) == 16)
        rc = bwd_scan_fit<T, NB, KP, 1>(a, fit, s);
    else
        rc = narrow(a.q.f, a.l) ? bwd_scan_fit<T, NB, KP, 1>(a, fit, s) : bwd_scan_fit<T, NB, KP, 2>(a, fit, s);
    if (rc) return rc;
    if (a.q.f.heads == a.q.f.heads_k) return fit ? grad_launch<T, NB, KP, true, false>(a, s) : grad_launch<T, NB, KP, false, false>(a, s);
    return fit ? grad_launch<T, NB, KP, true, true>(a, s) : grad_launch<T, NB, KP, false, true>(a, s);
}
template <typename T>
static int bwd_type(const BwdArgs& a, hipStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (planes_kept(a.q.f) == 2) return pad_k(a.q.f.dk) == 64 ? bwd_launch<T, 2, 64>(a, s) : bwd_launch<T, 2, 128>(a, s);
    return pad_k(a.q.f.dk) == 64 ? bwd_launch<T, 3, 64>(a, s) : bwd_launch<T, 3, 128>(a, s);
}

}  // namespace gd
}  // namespace vms

using namespace vms;

extern "C" int vms_gated_delta_bwd(const vms_gated_delta_bwd_params* qq, void* stream) {
    VMS_CHECK(qq != nullptr, "null params");
    if (int rc = gd::validate(qq->f)) return rc;
    VMS_CHECK(qq->f.for_backward, "the forward must have run with for_backward");
    VMS_CHECK(qq->dout_seq_stride > -(1LL << 31) && qq->dout_seq_stride < (1LL << 31), "strides along the sequence of less than 2^31 elements");
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
