// gated_delta_fwd.hip -- gated delta rule, forward (vms_gated_delta_fwd): the algebra and the layouts are in gated_delta.h.
//
//   gd_prep   one wave per (chunk, head): the gates, T (triangular inverse in fp32), M.
//   gd_scan   the walk over the chunks.  The columns of S (and of V, U, O) never meet: a workgroup owns 16 CT of them for the whole
//             sequence.  Four of its waves walk the chain and split the chunk's 64 tokens and S's dk rows: wave w computes token tile w of
//             K S0 and U and dk / 4 rows of S, which stay in its accumulators.  The other four load, make O and store.
#include <type_traits>

#include "gated_delta.h"

namespace vms {
namespace gd {

// g below this forgets everything (exp underflows) and would cost the cumulative sums their low bits
constexpr float kMinGate = -104.f;

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// ---- T, M and gates of one chunk -----------------------------------------------------------------------------
// Bound by bytes: (8, 8192, 8 heads, 128) bf16 reads 268 MB of q and k and writes 262 MB in 96 us, 5.5 TB/s (a large copy: 5.2); in calls with few
// chunks by one wave's chain of steps (10 us, bf16, 64).
// K K^T and Q K^T (16x16x32 bf16 MFMA, operands straight from memory), L from double cumulative sums (differences of long sums keep
// their bits), then T: the four 16 x 16 diagonal blocks by forward substitution (16 lanes each, a column per lane; a power series would
// lose ~13 bits to the binomials of equal keys), joined by T21 = -T22 A21 T11 with fp32 MFMA.
template <typename T, int KP, int FIT, int NB>
__global__ __launch_bounds__(64, 2) void gd_prep_kernel(const vms_gated_delta_params p, const Layout l) {
    constexpr int NX = Prec<T>::NX, NO = Prec<T>::NO;
    constexpr int AR = 68;   // row pitch of As, floats
    __shared__ __attribute__((aligned(16))) float As[C * AR];
    __shared__ __attribute__((aligned(32))) double Gs[C];
    __shared__ float bs[C];
    const int lane = threadIdx.x, n = lane & 15, q4 = lane >> 4;
    const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int len = length_of(p, b);
    if (c * C >= len) return;
    const int hk = h / (p.heads / p.heads_k);
    const int64_t slot = ((int64_t)b * p.heads + h) * l.chunks + c;
    char* const ws = static_cast<char*>(p.workspace);

    const Rows<T> Q(p.q, (int64_t)b * p.q_batch_stride + (int64_t)hk * p.q_head_stride, p.q_seq_stride, len, p.reverse);
    const Rows<T> K(p.k, (int64_t)b * p.k_batch_stride + (int64_t)hk * p.k_head_stride, p.k_seq_stride, len, p.reverse);
    auto rows = [&](const Rows<T>& x, int rt, int kb) __attribute__((always_inline)) {
        const int i = c * C + 16 * rt + n;
        return fit_load<FIT, T>(x.row(i < len ? i : len - 1), 32 * kb + 8 * q4, p.dk);
    };
    auto as_frag = [&](const Raw8<T>& r, int kb) __attribute__((always_inline)) { return planes_of<T>(fit_clear<FIT, T>(r, 32 * kb + 8 * q4, p.dk)); };
    Raw8<T> kraw[4][KP / 32];
#pragma unroll
    for (int rt = 0; rt < 4; ++rt)
#pragma unroll
        for (int kb = 0; kb < KP / 32; ++kb) kraw[rt][kb] = rows(K, rt, kb);
    // q's rows of the next 16 tokens are on their way while these are multiplied, k's and the first of q before the gates: a chunk is one wave, and each
    // memory latency it waits for shows in calls with few chunks
    constexpr bool kEarly = KP * (int)sizeof(T) <= 256;   // (two sets of fp32 rows of 128 would spill)
    Raw8<T> qraw[KP / 32], qnext[KP / 32];
#pragma unroll
    for (int kb = 0; kb < KP / 32; ++kb) qnext[kb] = rows(Q, 0, kb);

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
        G *= 1.4426950408889634;   // exponents of 2 from here on
        const double last = __shfl(G, 63);
        Gs[lane] = G;
        bs[lane] = be;
        Gates* const o = reinterpret_cast<Gates*>(ws + l.gates) + slot;
        o->gam[lane] = fast_exp2((float)G);
        o->bet[lane] = be;
        o->del[lane] = fast_exp2((float)(last - G));
        o->G[lane] = G;
    }
    __syncthreads();

    char* const tw = ws + l.tri + slot * l.tri_slot;
    char* const mw = tw + NS * kTri;
    char* const ttw = mw + NO * kTri;   // transposes (for_backward)
    char* const mtw = ttw + NB * kTri;
    auto put4 = [&](char* at, const f32x4& v) __attribute__((always_inline)) {   // half an operand, NB planes
        float x[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
        Frag<NB ? NB : 1> f;
        split<NB ? NB : 1>(x, f);
#pragma unroll
        for (int i2 = 0; i2 < NB; ++i2) *reinterpret_cast<bf16x4*>(at + i2 * kTri) = __builtin_shufflevector(f.p[i2], f.p[i2], 0, 1, 2, 3);
    };
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
        f32x4 kk[4], qk[4], kq[4];   // kq: Q K^T once more, lanes along j: the transpose of M
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) { kk[ct] = f32x4{0.f, 0.f, 0.f, 0.f}; qk[ct] = kk[ct]; kq[ct] = kk[ct]; }
#pragma unroll
        for (int kb = 0; kb < KP / 32; ++kb) {
            if (!kEarly && rt > 0) qnext[kb] = rows(Q, rt, kb);
            qraw[kb] = qnext[kb];
            if (kEarly && rt < 3) qnext[kb] = rows(Q, rt + 1, kb);
        }
#pragma unroll
        for (int kb = 0; kb < KP / 32; ++kb) {
            const Frag<NX> qi = as_frag(qraw[kb], kb), ki = as_frag(kraw[rt][kb], kb);
#pragma unroll
            for (int ct = 0; ct <= rt; ++ct) {   // [j][i]: lane i, 4 consecutive j
                const Frag<NX> kj = ct == rt ? ki : as_frag(kraw[ct][kb], kb);
                mma<NS>(kk[ct], kj, ki);
                mma<NO>(qk[ct], kj, qi);
                if constexpr (NB > 0) mma<NB>(kq[ct], qi, kj);
            }
        }
        const int i = 16 * rt + n;
        const double Gi = Gs[i];
        const float bi = bs[i];
#pragma unroll
        for (int ct = 0; ct <= rt; ++ct) {
            f32x4 a;
            const f64x4 Gj = *reinterpret_cast<const f64x4*>(&Gs[16 * ct + 4 * q4]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = 16 * ct + 4 * q4 + r;
                const float L = decay(j <= i, Gi - Gj[r]);
                const float x = bi * L * kk[ct][r], y = p.scale * L * qk[ct][r];
                a[r] = j < i ? x : 0.f;
                qk[ct][r] = j <= i ? y : 0.f;
            }
            *reinterpret_cast<f32x4*>(&As[i * AR + 16 * ct + 4 * q4]) = a;
            if constexpr (NB > 0) {
                const int j = 16 * ct + n;
                const double Gn = Gs[j];
                const f64x4 G4 = *reinterpret_cast<const f64x4*>(&Gs[16 * rt + 4 * q4]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i2 = 16 * rt + 4 * q4 + r;
                    const float x = p.scale * decay(j <= i2, G4[r] - Gn) * kq[ct][r];
                    kq[ct][r] = j <= i2 ? x : 0.f;
                }
                put4(mtw + 1024 * tri_t(ct, rt >> 1) + 16 * lane + 8 * (rt & 1), kq[ct]);
            }
        }
        if (NB > 0 && (rt & 1) == 0) put4(mtw + 1024 * tri_t(rt + 1, rt >> 1) + 16 * lane, f32x4{0.f, 0.f, 0.f, 0.f});   // above the diagonal
#pragma unroll
        for (int kb = 0; kb <= rt / 2; ++kb) {
            const Frag<NO> f = frag_of<NO>(qk[2 * kb], qk[2 * kb + 1]);
#pragma unroll
            for (int i2 = 0; i2 < NO; ++i2)
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
    if constexpr (NB > 0) {
#pragma unroll
        for (int ct = 0; ct < 4; ++ct)
#pragma unroll
            for (int ib = ct / 2; ib < 2; ++ib)
#pragma unroll
                for (int half = 0; half < 2; ++half) put4(ttw + 1024 * tri_t(ct, ib) + 16 * lane + 8 * half, 2 * ib + half >= ct ? b_of(2 * ib + half, ct) : zero);
    }
}

// ---- the walk over the chunks --------------------------------------------------------------------------------
// What bounds it is the chain of one chunk (K S0 -> R -> U -> S1), not a rate: a head is 16 .. 64 tokens of work per step on one CU.  (8, 8192, 8 heads,
// 128 x 128) bf16, 378 us: 2.95 us or 5800 cycles per chunk, of which the matrix cores work 1460 and LDS 3820: S0's planes are read by eight waves (three by the chain, two
// by the others) and handed over three times, and 1680 cycles go to bank conflicts (rows of K's tile, whose pitch suits the transposing reads, 8-byte writes of the
// exchanges, V's tile).  Steps that led here, same sizes, us per chunk:
//   a wave with a whole chunk of 16 columns to itself, every wave reading all of K, Q, T, M from LDS             5.4
//   four waves on one chunk, K, Q, T, M straight from memory, a chunk ahead                                      2.4
//   four waves on the chain, four on loads and outputs; lines instead of operands from memory                    2.05
//   three planes on the chain instead of two, two instead of one in the outputs (for their accuracy)             2.95
// Lines: an operand's lanes are 16 rows x 4 pieces of 16 bytes with neighbouring lanes in different rows, and the memory pipe then takes 64 accesses
// for a load of 1 KB instead of 16 (2825 of a chunk's 5100 cycles).  Read as lines, through LDS into operands, K also stands there for its transpose.  Asked
// for two chunks ahead (one chunk is less than a loaded memory's latency) and spread over the phases: a wave stands still while the pipe is full.
template <typename T, int KP, int CT, int FIT, int NB>
struct ScanLds {   // bytes and places in LDS
    static constexpr int NX = Prec<T>::NX, NU = NB > Prec<T>::NO ? NB : Prec<T>::NO;   // planes of U: what M U and the backward need
    static constexpr int kK = NX * tile_bytes<KP>(), kPiece = VTile<T, CT, FIT != 0>::kBytes, kQRow = KP * (int)sizeof(T) + 16;
    static constexpr int kRest = Exchange<NS, CT, KP>::kBytes + 2 * Exchange<NS, CT, C>::kBytes + Exchange<NU, CT, C>::kBytes + 3 * 4 * kPiece + 2 * 4 * GateTile::kBytes;
    static constexpr bool kStaged = 2 * kK + kRest + 4 * 16 * kQRow <= 163840;   // K and Q come through LDS; with many planes two tiles do not fit
    static constexpr int kQ = kStaged ? 16 * kQRow : 0;   // per wave
    static constexpr int S = (kStaged ? 2 : 1) * kK, R = S + Exchange<NS, CT, KP>::kBytes, U = R + Exchange<NS, CT, C>::kBytes, D = U + Exchange<NU, CT, C>::kBytes,
                         V = D + Exchange<NS, CT, C>::kBytes,           // V, O: one and one per wave and buffer
                         G = V + 3 * 4 * kPiece, Q = G + 2 * 4 * GateTile::kBytes, kBytes = Q + 4 * kQ;
    static_assert(kBytes <= 163840, "160 KB of LDS");
};

template <typename T, int KP, int CT, int FIT, int NB>
__global__ __launch_bounds__(512, 1) void gd_scan_kernel(const vms_gated_delta_params p, const Layout l, const int slices) {
    constexpr int NX = Prec<T>::NX, NO = Prec<T>::NO;
    constexpr int KB = KP / 32, DW = KP / 64;   // 32-column blocks of k; 16-row tiles of S per wave
    constexpr bool WHOLE = FIT != 0;
    using Lds = ScanLds<T, KP, CT, FIT, NB>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const Exchange<NS, CT, KP> Sx{lds + Lds::S};
    const Exchange<NS, CT, C> Rx{lds + Lds::R}, Dx{lds + Lds::D};   // R, del U
    const Exchange<Lds::NU, CT, C> Ux{lds + Lds::U};

    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, q4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), w = wave & 3;
    int pair, slice;
    pair_of(blockIdx.x, p.batch * p.heads, slices, pair, slice);
    const int b = pair / p.heads, h = pair % p.heads, hk = h / (p.heads / p.heads_k);
    const int len = length_of(p, b), nc = (len + C - 1) / C;
    const int col0 = slice * CT * 16;
    char* const ws = static_cast<char*>(p.workspace);
    const int64_t slot0 = (int64_t)pair * l.chunks;
    const Rows<T> K(p.k, (int64_t)b * p.k_batch_stride + (int64_t)hk * p.k_head_stride, p.k_seq_stride, len, p.reverse);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    auto tile = [&](int odd) __attribute__((always_inline)) { return lds + (Lds::kStaged ? odd * Lds::kK : 0); };
    auto v_at = [&](int odd) __attribute__((always_inline)) { return lds + Lds::V + (4 * odd + w) * Lds::kPiece; };
    auto g_at = [&](int odd) __attribute__((always_inline)) { return reinterpret_cast<float*>(lds + Lds::G + (4 * odd + w) * GateTile::kBytes); };
    auto fetch_rows = [&](const Rows<T>& x, int c, Raw8<T> (&r)[KB]) __attribute__((always_inline)) {   // operands: token 16 w + n
        const int at = c * C + 16 * w + n;
        const T* const row = x.row(at < len ? at : len - 1);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) r[kb] = fit_load<FIT, T>(row, 32 * kb + 8 * q4, p.dk);
    };
    // the same 16 rows by lines: piece i of 8 columns
    auto piece_row = [&](int i) __attribute__((always_inline)) { return (lane + 64 * i) / (KP / 8); };
    auto piece_col = [&](int i) __attribute__((always_inline)) { return 8 * ((lane + 64 * i) % (KP / 8)); };
    auto fetch_lines = [&](const Rows<T>& x, int c, Raw8<T> (&r)[KB]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KB; ++i) {
            const int at = c * C + 16 * w + piece_row(i);
            r[i] = fit_load<FIT, T>(x.row(at < len ? at : len - 1), piece_col(i), p.dk);
        }
    };
    // Both sides below meet at three barriers per chunk: S is there; R is there; U is there.  Loads are asked for two chunks ahead.
    if (wave < 4) {
        // ---- the chain: U, S
        __builtin_amdgcn_s_setprio(2);   // the other wave of this SIMD has slack
        f32x4 S[DW][CT];   // rows 16 (DW w + d) + 4 q4 + r, column n
        const int64_t sbase = (int64_t)pair * p.dk * p.dv;
#pragma unroll
        for (int d = 0; d < DW; ++d)
#pragma unroll
            for (int j = 0; j < CT; ++j) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * (DW * w + d) + 4 * q4 + r, col = col0 + col_of<CT>(j, n);
                    S[d][j][r] = p.initial_state && row < p.dk && col < p.dv ? p.initial_state[sbase + (int64_t)row * p.dv + col] : 0.f;
                }
                Sx.put(j, n, 16 * (DW * w + d) + 4 * q4, S[d][j]);
            }
        auto fetch_t = [&](int c, Frag<NS> (&t)[2]) __attribute__((always_inline)) {   // rows 16 w + n of T (blocks 0, 1; tiles 0 and 1 have no block 1)
            const char* const at = ws + l.tri + (slot0 + c) * l.tri_slot;
            t[0] = tri_rows<NS>(at, w, 0, lane);
            t[1] = tri_rows<NS>(at, w, w >= 2 ? 1 : 0, lane);
        };
        Raw8<T> kr[KB];
        auto chunk = [&](int c, auto odd_c, Frag<NS> (&tf)[2]) __attribute__((always_inline)) {
            constexpr int odd = decltype(odd_c)::value;
            char* const Ks = tile(odd);
            VTile<T, CT, WHOLE> vt;
            vt.base = v_at(odd);
            GateTile gt;
            gt.base = g_at(odd);
            __syncthreads();   // S is there; (not staged) K's tile is no longer read
            f32x4 P[CT];   // K S0
#pragma unroll
            for (int j = 0; j < CT; ++j) P[j] = zero;
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
                for (int j = 0; j < CT; ++j) mma<NS>(P[j], kf, Sx.get(j, n, 32 * kb + 8 * q4));
            }
            if constexpr (!Lds::kStaged) fetch_rows(K, c + 1 < nc ? c + 1 : c, kr);
            const f32x4 ga = gt.four(0, q4), be = gt.four(1, q4), de = gt.four(2, q4);
            const float glast = gt.last();
            f32x4 vv[CT];
#pragma unroll
            for (int j = 0; j < CT; ++j) vv[j] = vt.get(j, n, q4);
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                f32x4 R;
#pragma unroll
                for (int r = 0; r < 4; ++r) R[r] = be[r] * fmaf(-ga[r], P[j][r], vv[j][r]);   // beta = 0 behind the end
                Rx.put(j, n, paired(w, q4), R);
            }
            __syncthreads();
            f32x4 U[CT];   // T R
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                U[j] = zero;
                mma<NS>(U[j], tf[0], Rx.get(j, n, 8 * q4));
            }
            if (w >= 2) {
#pragma unroll
                for (int j = 0; j < CT; ++j) mma<NS>(U[j], tf[1], Rx.get(j, n, 32 + 8 * q4));
                settle(U);
            }
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                const f32x4 x = U[j] * de;
                Dx.put(j, n, paired(w, q4), x);
                Ux.put(j, n, paired(w, q4), U[j]);
            }
            __syncthreads();
            // S1 = gam S0 + K^T (del U)
#pragma unroll
            for (int d = 0; d < DW; ++d)
#pragma unroll
                for (int j = 0; j < CT; ++j) S[d][j] *= glast;
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                Frag<NS> uf[CT];
#pragma unroll
                for (int j = 0; j < CT; ++j) uf[j] = Dx.get(j, n, 32 * tb + 8 * q4);
#pragma unroll
                for (int d = 0; d < DW; ++d) {
                    const Frag<NX> kc = tile_cols<KP, NX>(Ks, DW * w + d, tb, n, q4);
#pragma unroll
                    for (int j = 0; j < CT; ++j) mma<NS>(S[d][j], kc, uf[j]);
                }
            }
#pragma unroll
            for (int d = 0; d < DW; ++d)
#pragma unroll
                for (int j = 0; j < CT; ++j) Sx.put(j, n, 16 * (DW * w + d) + 4 * q4, S[d][j]);
            fetch_t(c + 2 < nc ? c + 2 : nc - 1, tf);
        };
        if (nc > 0) {
            Frag<NS> t0[2], t1[2];
            if constexpr (!Lds::kStaged) fetch_rows(K, 0, kr);
            fetch_t(0, t0);
            fetch_t(nc > 1 ? 1 : 0, t1);
            for (int c = 0;;) {
                chunk(c, std::integral_constant<int, 0>{}, t0);
                if (++c == nc) break;
                chunk(c, std::integral_constant<int, 1>{}, t1);
                if (++c == nc) break;
            }
        }
        if (p.final_state) {
#pragma unroll
            for (int d = 0; d < DW; ++d)
#pragma unroll
                for (int j = 0; j < CT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = 16 * (DW * w + d) + 4 * q4 + r, col = col0 + col_of<CT>(j, n);
                        if (row < p.dk && col < p.dv) p.final_state[sbase + (int64_t)row * p.dv + col] = S[d][j][r];
                    }
        }
    } else {
        // ---- the outputs (O, and S0 and U for the backward), and what both sides read
        const Rows<T> Q(p.q, (int64_t)b * p.q_batch_stride + (int64_t)hk * p.q_head_stride, p.q_seq_stride, len, p.reverse);
        const Rows<T> V(p.v, (int64_t)b * p.v_batch_stride + (int64_t)h * p.v_head_stride, p.v_seq_stride, len, p.reverse);
        const Rows<T> O_(p.out, (int64_t)b * p.out_batch_stride + (int64_t)h * p.out_head_stride, p.out_seq_stride, len, p.reverse);
        const Gates* const gates = reinterpret_cast<const Gates*>(ws + l.gates) + slot0;
        char* const Qs = lds + Lds::Q + w * Lds::kQ;
        struct Ahead {
            Raw8<T> k[KB], q[KB];   // token 16 w + n, or its lines
            VTile<T, CT, WHOLE> v;
            GateTile g;
        };
        auto fetch_m = [&](int c, Frag<NO> (&m)[2]) __attribute__((always_inline)) {   // rows 16 w + n of M
            const char* const at = ws + l.tri + (slot0 + c) * l.tri_slot + NS * kTri;
            m[0] = tri_rows<NO>(at, w, 0, lane);
            m[1] = tri_rows<NO>(at, w, w >= 2 ? 1 : 0, lane);
        };
        auto fetch_q = [&](int c, Ahead& a) __attribute__((always_inline)) {
            if constexpr (Lds::kStaged) fetch_lines(Q, c, a.q);
        };
        auto fetch_k = [&](int c, Ahead& a) __attribute__((always_inline)) {
            if constexpr (Lds::kStaged) fetch_lines(K, c, a.k);
        };
        auto fetch_v = [&](int c, Ahead& a) __attribute__((always_inline)) {
            a.v.fetch(V, c * C + 16 * w, len, col0, p.dv, lane);
            a.g.fetch(reinterpret_cast<const float*>(gates + c), w, lane);
        };
        auto hand = [&](int c, auto odd_c, Ahead& a) __attribute__((always_inline)) {   // into LDS; Q, V's and the gates' places are this wave's and its twin's
            constexpr int odd = decltype(odd_c)::value;
            if constexpr (Lds::kStaged) {
#pragma unroll
                for (int i = 0; i < KB; ++i) {
                    tile_put<KP, NX>(tile(odd), 16 * w + piece_row(i), piece_col(i), planes_of<T>(fit_clear<FIT, T>(a.k[i], piece_col(i), p.dk)));
                    const Raw8<T> x = fit_clear<FIT, T>(a.q[i], piece_col(i), p.dk);
                    __builtin_memcpy(__builtin_assume_aligned(Qs + piece_row(i) * Lds::kQRow + piece_col(i) * (int)sizeof(T), 16), &x, sizeof(x));
                }
            }
            a.v.base = v_at(odd);
            a.g.base = g_at(odd);
            a.v.hand(c * C + 16 * w, len, col0, p.dv, lane, true);
            a.g.hand(lane);
        };
        const OTile<T, CT, WHOLE> ot{v_at(2)};
        Raw8<T> qr[KB];
        auto chunk = [&](int c, auto odd_c, Ahead& mine, Ahead& other, Frag<NO> (&mf)[2]) __attribute__((always_inline)) {   // other: of chunk c + 1
            constexpr int odd = decltype(odd_c)::value;
            const int64_t slot = slot0 + c;
            __syncthreads();
            if (c > 0) ot.store(O_, (c - 1) * C + 16 * w, len, col0, p.dv, lane);
            const float sg = p.scale * g_at(odd)[n];
            f32x4 O[CT];   // S0^T Q^T, [v][token]: a lane holds 4 consecutive v
#pragma unroll
            for (int j = 0; j < CT; ++j) O[j] = zero;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                Raw8<T> x;
                if constexpr (Lds::kStaged) __builtin_memcpy(&x, __builtin_assume_aligned(Qs + n * Lds::kQRow + (32 * kb + 8 * q4) * (int)sizeof(T), 16), sizeof(x));
                else x = fit_clear<FIT, T>(qr[kb], 32 * kb + 8 * q4, p.dk);
                const Frag<NX> qf = planes_of<T>(x);
#pragma unroll
                for (int j = 0; j < CT; ++j) mma<NO>(O[j], Sx.template get<NO>(j, n, 32 * kb + 8 * q4), qf);
            }
            if constexpr (NB > 0) {
                if (w < KB) {   // S0, 32 rows per wave
                    Frag<NB> sf[CT];
#pragma unroll
                    for (int j = 0; j < CT; ++j) sf[j] = Sx.template get<NB>(j, n, 32 * w + 8 * q4);
                    store_frag<NB, CT, false>(ws + l.S0 + slot * l.s_slot, KP, l.vpad, 32 * w, 0, col0, sf, n, q4);
                }
            }
            if constexpr (!Lds::kStaged) fetch_rows(Q, c + 1 < nc ? c + 1 : c, qr);
            fetch_k(c + 2 < nc ? c + 2 : nc - 1, mine);
            __syncthreads();
            hand(c + 1, std::integral_constant<int, 1 - odd>{}, other);
            const int next = c + 3 < nc ? c + 3 : nc - 1;
            fetch_v(next, other);
            __syncthreads();
            fetch_q(next, other);
#pragma unroll
            for (int j = 0; j < CT; ++j) O[j] *= sg;
            // O += M U
            Frag<Lds::NU> uf[CT];
#pragma unroll
            for (int j = 0; j < CT; ++j) uf[j] = Ux.get(j, n, 8 * q4);
#pragma unroll
            for (int j = 0; j < CT; ++j) mma<NO>(O[j], uf[j], mf[0]);
            if (w >= 2) {
#pragma unroll
                for (int j = 0; j < CT; ++j) uf[j] = Ux.get(j, n, 32 + 8 * q4);
#pragma unroll
                for (int j = 0; j < CT; ++j) mma<NO>(O[j], uf[j], mf[1]);
                settle(O);
            }
            fetch_m(c + 2 < nc ? c + 2 : nc - 1, mf);
            ot.put(O, lane);
            if constexpr (NB > 0) store_frag<NB, CT, true>(ws + l.U + slot * l.u_slot, C, l.vpad, 16 * w, w & 1, col0, uf, n, q4);
        };
        if (nc > 0) {
            Ahead a0, a1;
            Frag<NO> m0[2], m1[2];
            if constexpr (!Lds::kStaged) fetch_rows(Q, 0, qr);
            auto fetch = [&](int c, Ahead& a) __attribute__((always_inline)) { fetch_k(c, a); fetch_v(c, a); fetch_q(c, a); };
            fetch(0, a0);
            fetch(nc > 1 ? 1 : 0, a1);
            fetch_m(0, m0);
            fetch_m(nc > 1 ? 1 : 0, m1);
            hand(0, std::integral_constant<int, 0>{}, a0);
            fetch_v(nc > 2 ? 2 : nc - 1, a0);
            fetch_q(nc > 2 ? 2 : nc - 1, a0);
            for (int c = 0;;) {
                chunk(c, std::integral_constant<int, 0>{}, a0, a1, m0);
                if (++c == nc) break;
                chunk(c, std::integral_constant<int, 1>{}, a1, a0, m1);
                if (++c == nc) break;
            }
            ot.store(O_, (nc - 1) * C + 16 * w, len, col0, p.dv, lane);
        }
        // padding behind the sequence's end
        T* const ob = static_cast<T*>(p.out) + (int64_t)b * p.out_batch_stride + (int64_t)h * p.out_head_stride;
        const int cn = p.dv - col0 < CT * 16 ? p.dv - col0 : CT * 16;
        for (int t = len + w; t < p.seqlen; t += 4)
            for (int cc = lane; cc < cn; cc += 64) ob[(int64_t)t * p.out_seq_stride + col0 + cc] = static_cast<T>(0.f);
    }
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
    // the walks' launches of 512 threads have to stay below 2^32 threads (fewer columns than these only where workgroups are few)
    const int least = p.for_backward ? bwd_columns(p.dtype, planes_kept(p), pad_k(p.dk)) : 32;
    VMS_CHECK((int64_t)p.batch * p.heads * (ceil_to(p.dv, 32) / least) < (1LL << 32) / 512, "problem too large");
    VMS_CHECK(p.q && p.k && p.v && p.g && p.beta, "q, k, v, g, beta are required");
    for (const int64_t n : {p.q_seq_stride, p.k_seq_stride, p.v_seq_stride, p.out_seq_stride})
        VMS_CHECK(n > -(1LL << 31) && n < (1LL << 31), "strides along the sequence of less than 2^31 elements");
    const Layout l = layout(p);
    VMS_CHECK(p.workspace != nullptr && p.workspace_bytes >= l.bytes, "workspace is too small (vms_gated_delta_workspace_bytes)");
    VMS_CHECK((reinterpret_cast<uintptr_t>(p.workspace) & 15) == 0, "workspace must be 16-byte aligned");
    return VMS_OK;
}

template <typename T, int KP, int CT, int FIT, int NB>
static int scan_launch(const vms_gated_delta_params& p, const Layout& l, hipStream_t s) {
    constexpr int lds = ScanLds<T, KP, CT, FIT, NB>::kBytes;
    static PerDeviceOnce once;
    if (int rc = allow_lds(once, reinterpret_cast<const void*>(&gd_scan_kernel<T, KP, CT, FIT, NB>), lds)) return rc;
    const int slices = (l.vpad + CT * 16 - 1) / (CT * 16);
    hipLaunchKernelGGL((gd_scan_kernel<T, KP, CT, FIT, NB>), dim3(p.batch * p.heads * slices), dim3(512), lds, s, p, l, slices);
    VMS_LAUNCH_CHECK();
    return VMS_OK;
}
template <typename T, int KP, int FIT, int NB>
static int fwd_launch(const vms_gated_delta_params& p, hipStream_t s) {
    const Layout l = layout(p);
    hipLaunchKernelGGL((gd_prep_kernel<T, KP, FIT, NB>), dim3(l.chunks, p.heads, p.batch), dim3(64), 0, s, p, l);
    VMS_LAUNCH_CHECK();
    return narrow(p, l) ? scan_launch<T, KP, 1, FIT, NB>(p, l, s) : scan_launch<T, KP, 2, FIT, NB>(p, l, s);
}
template <typename T, int KP, int FIT>
static int fwd_train(const vms_gated_delta_params& p, hipStream_t s) {
        if (!p.for_backward) return fwd_launch<T, KP, FIT, 0>(p, s);
    if constexpr (sizeof(T) == 2)
        if (planes_kept(p) == 2) return fwd_launch<T, KP, FIT, 2>(p, s);
    return fwd_launch<T, KP, FIT, 3>(p, s);
}
template <typename T, int KP>
static int fwd_fit(const vms_gated_delta_params& p, hipStream_t s) {
    switch (fit_of(p.dk, p.dv)) {
        case 2: return fwd_train<T, KP, 2>(p, s);
        case 1: return fwd_train<T, KP, 1>(p, s);
        default: return fwd_train<T, KP, 0>(p, s);
    }
}
template <typename T>
static int fwd_type(const vms_gated_delta_params& p, hipStream_t s) {
    return pad_k(p.dk) == 64 ? fwd_fit<T, 64>(p, s) : fwd_fit<T, 128>(p, s);
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
