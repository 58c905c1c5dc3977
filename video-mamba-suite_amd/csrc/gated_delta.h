// gated_delta.h -- what the gated delta rule's kernels share (gated_delta_fwd.hip, gated_delta_bwd.hip): the chunk's
// algebra, operand precision, fragment layouts and the workspace they pass from kernel to kernel.
//
// Per batch entry and head, S (dk x dv), a_t = exp(g_t):
//   S' = a_t S_{t-1};  e_t = v_t - S'^T k_t;  u_t = beta_t e_t;  S_t = S' + k_t u_t^T;  o_t = scale S_t^T q_t
// over 64 tokens at once (G = cumulative sum of g inside the chunk, gam = exp(G), del = exp(G_63 - G), L_ij = exp(G_i - G_j)):
//   N_ij = L_ij k_i.k_j (i > j);  T = (I + diag(beta) N)^-1;  M_ij = scale L_ij q_i.k_j (i >= j)
//   U = T beta (V - gam K S0);  O = scale gam Q S0 + M U;  S1 = gam_63 S0 + K^T (del U)
// T, M and the gates depend on no state: one parallel launch makes them for every chunk; what is left for the sequential walk
// over the chunks is four products per chunk.
//
// Precision.  Everything runs on the bf16 matrix cores with fp32 accumulators.  An operand is the sum of 1 .. 3 bf16 planes
// (8 bits of the significand each: off by at most 2^-8, 2^-16, 2^-24 of itself), so that
//   inputs are exact:                                                          bf16 1 plane, fp16 2, fp32 3                     (NX)
//   the state's recurrence in the forward (T, R, U, S as operands):            3, since final states are fp32 whatever the inputs are  (NS)
//   what enters 16-bit outputs alone (M, U and S0 as their operands):          2, 3 for fp32                                    (NO)
//   what the backward computes and reads of the forward (S0, U, dS1, Y, ...):  3 for fp32 inputs and where a state comes in or goes out: its gradient and
//     those of fp32 gates are fp32 then; else 2                                                                                  (NB)
// Not 1 for bf16 anywhere: outputs and gradients are differences of larger terms where keys share a direction, and a plane's 2^-8 in M, U
// or Y shows 5 to 20 times as large as the result's own rounding (1.7e-3).  Relative error in the norm before that rounding, the algebra above in 64
// bits with its operands rounded, 512 tokens, bf16, 64 x 64, keys of cosine 0.99 and beta 1 (independent keys, random beta):
//   one plane of M, S0, U, dS1, Y, else two   out 9.1e-3 (1.7e-3), dq 7.5e-3 (1.7e-3), dg 3.8e-2 (1.9e-3), final state 2.3e-5 (3.7e-6)
//   two throughout                            out 3.0e-5 (5.2e-6), dq 1.8e-5 (4.5e-6), dg 5.8e-4 (5.4e-6), final state 2.3e-5 (3.7e-6)
//   three throughout                          out 3.0e-7 (5.8e-8), dq 2.5e-7 (6.3e-8), dg 7.1e-6 (1.6e-7), final state 3.4e-7 (5.4e-8)
// Calls of bf16, us: (8, 8192, 8 heads, 128 x 128) 309, 353, 477 (428 with the planes above); training at (8, 3136, 6 heads, 128 x 128) 416, 613, 969
// (640; with an initial state 909).
#pragma once
#include "vms_common.h"

namespace vms {
namespace gd {

constexpr int C = 64;   // tokens of a chunk

using bf16x8 = vec_t<bf16_t, 8>;
using bf16x4 = vec_t<bf16_t, 4>;
using f32x4 = vec_t<float, 4>;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

template <typename T> struct Prec;
constexpr int NS = 3;   // (NB is a parameter of the kernels: planes_kept)
template <> struct Prec<bf16_t> { static constexpr int NX = 1, NO = 2; };
template <> struct Prec<f16_t> { static constexpr int NX = 2, NO = 2; };
template <> struct Prec<float> { static constexpr int NX = 3, NO = 3; };

// An operand of v_mfma_f32_16x16x32_bf16: lane = 16 p + n holds row (A) / column (B) n and 8 of the 32 contracted indices.
// Two index orders are in use (any order is right as long as both operands share it):
//   natural   element e of quarter p = index 8 p + e          (16-byte reads of a row)
//   paired    e < 4: 4 p + e, else 16 + 4 p + (e - 4)          (the accumulators of two 16-row tiles ARE the operand:
//                                                               a product's result enters the next product without moving)
template <int N> struct Frag { bf16x8 p[N]; };

template <int KEEP, int NA, int NB>
__device__ __forceinline__ void mma(f32x4& acc, const Frag<NA>& a, const Frag<NB>& b) {
#pragma unroll
    for (int s = KEEP - 1; s >= 0; --s)   // the smallest products first
#pragma unroll
        for (int i = 0; i <= s; ++i)
            if (i < NA && s - i < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[s - i], acc, 0, 0, 0);
}

// Results of products in a block that not every wave enters, at the end of the block: a matrix instruction's result may be touched 8 wait states after it at the earliest,
// and the compiler's count of them misses ways through short conditional blocks (tools/isa_hazards.py --mfma).  The empty statements hold the results
// here, in the order of these statements; behind the last one the waits are over.
__device__ __forceinline__ void settle(f32x4& x) { asm volatile("s_nop 7" : "+v"(x)); }
template <int N, typename... Rest>
__device__ __forceinline__ void settle(f32x4 (&x)[N], Rest&... rest) {
#pragma unroll
    for (int i = 0; i < (sizeof...(rest) ? N : N - 1); ++i) asm volatile("" : "+v"(x[i]));
    if constexpr (sizeof...(rest) > 0) settle(rest...);
    else settle(x[N - 1]);
}

// x0, x1 -> their bf16 values (round to nearest) in one register; what is left of them
__device__ __forceinline__ unsigned take_bf16(float& x0, float& x1, bool last) {
    using bf16x2 = vec_t<bf16_t, 2>;
    const bf16x2 h = {static_cast<bf16_t>(x0), static_cast<bf16_t>(x1)};
    const unsigned u = __builtin_bit_cast(unsigned, h);
    if (!last) {
        x0 -= __builtin_bit_cast(float, u << 16);
        x1 -= __builtin_bit_cast(float, u & 0xffff0000u);
    }
    return u;
}
// x -> N bf16 planes whose sum is x up to 2^-8N of itself
template <int N>
__device__ __forceinline__ void split(float (&x)[8], Frag<N>& f) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        vec_t<unsigned, 4> u;
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = take_bf16(x[2 * e], x[2 * e + 1], i + 1 == N);
        f.p[i] = __builtin_bit_cast(bf16x8, u);
    }
}
template <int N>
__device__ __forceinline__ Frag<N> frag_of(const f32x4& a, const f32x4& b) {   // two 16-row tiles, paired order
    float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    Frag<N> f;
    split<N>(x, f);
    return f;
}

__device__ __forceinline__ bf16x4 read_tr(const char* at) {   // 4 x 16 elements transposed among 16 lanes
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(at));
}
__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// 8 elements of a row as they stand in memory: columns c .. c+7 of a row of n, any alignment.  WHOLE: n % 8 == 0, one 16- or 32-byte load;
// otherwise element by element.  Never a branch: what lies outside is read from a place that exists and becomes zero in clear(), when it is
// used.  (Behind a branch the loads of the next chunk meet the other side's values in a register copy, which waits for them at once.)
template <typename T> struct Raw8 { T v[8]; };
template <bool WHOLE, typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* row, int c, int n) {
    Raw8<T> r;
    if constexpr (WHOLE) {
        __builtin_memcpy(&r, row + (c < n ? c : 0), sizeof(r));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r.v[e] = row[c + e < n ? c + e : 0];
    }
    return r;
}
template <bool WHOLE, typename T>
__device__ __forceinline__ Raw8<T> clear(Raw8<T> r, int c, int n, bool ok) {   // ok: the row exists
    if constexpr (WHOLE) {
        unsigned w[sizeof(r) / 4];
        __builtin_memcpy(w, &r, sizeof(r));
#pragma unroll
        for (int i = 0; i < (int)(sizeof(r) / 4); ++i) w[i] = ok && c < n ? w[i] : 0u;
        __builtin_memcpy(&r, w, sizeof(r));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r.v[e] = ok && c + e < n ? r.v[e] : static_cast<T>(0.f);
    }
    return r;
}
// The rows of q and k in the order of the walk.  FIT says how dk meets the tile: 0 any, 1 dk % 8 == 0, 2 dk == KP (nothing to clear).  Rows behind the end
// are the last row again: beta = 0 and the triangles keep them out of everything (gd_prep, the walks).
template <typename T>
struct Rows {
    const T* first;   // token 0 of the walk
    int step;         // elements to the next one (strides of 2^31 and more are refused)
    __device__ __forceinline__ Rows(const void* base, int64_t batch_head, int64_t seq_stride, int len, int reverse) {
        first = static_cast<const T*>(base) + batch_head + (reverse && len > 0 ? (int64_t)(len - 1) * seq_stride : 0);
        step = reverse ? -(int)seq_stride : (int)seq_stride;
    }
    __device__ __forceinline__ const T* row(int i) const { return first + (int64_t)i * step; }
};
template <int FIT, typename T>
__device__ __forceinline__ Raw8<T> fit_load(const T* row, int c, int n) {
    if constexpr (FIT == 2) {
        Raw8<T> r;
        __builtin_memcpy(&r, row + c, sizeof(r));
        return r;
    } else {
        return load_raw8<FIT == 1, T>(row, c, n);
    }
}
template <int FIT, typename T>
__device__ __forceinline__ Raw8<T> fit_clear(const Raw8<T>& r, int c, int n) {
    if constexpr (FIT == 2) return r;
    else return clear<FIT == 1, T>(r, c, n, true);
}
inline int fit_of(int dk, int dv) { return dv % 8 || dk % 8 ? 0 : dk == 64 || dk == 128 ? 2 : 1; }

// Columns of a walk's CT tiles: lane n of tile j has column 4 CT (n / 4) + 4 j + n % 4, so that the 4 CT columns a lane holds of a transposed product
// (rows 4 p + r of the CT tiles) stand side by side in memory: one store of 16 bytes instead of two of 8.
template <int CT> __device__ __forceinline__ int col_of(int j, int n) { return 4 * CT * (n >> 2) + 4 * j + (n & 3); }

// A wave's 16 tokens x 16 CT columns of v (or of out's gradient), through LDS into accumulator layout (tokens 4 p + r, column col_of(j, n)): one
// load of whole 16-byte pieces and a transposing read instead of 4 CT loads of single elements, each of which costs the memory pipe 30 cycles.
template <typename T, int CT, bool WHOLE>
struct VTile {
    static constexpr int kRow = 16 * CT * (int)sizeof(T) + 16, kBytes = 16 * kRow;   // per wave
    static constexpr int kPieces = 16 * CT * 2, kN = (kPieces + 63) / 64;             // pieces of 8 elements
    char* base;
    Raw8<T> r[kN];
    __device__ __forceinline__ void fetch(const Rows<T>& x, int first, int len, int col0, int dv, int lane) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int id = lane + 64 * i, row = (id / (2 * CT)) & 15, at = first + row;
            r[i] = load_raw8<WHOLE, T>(x.row(at < len ? at : len - 1), col0 + 8 * (id % (2 * CT)), dv);
        }
    }
    // rows behind the end: kept (v, whose beta is 0) or cleared (gradients)
    __device__ __forceinline__ void hand(int first, int len, int col0, int dv, int lane, bool keep_tail) const {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int id = lane + 64 * i, row = id / (2 * CT);
            const Raw8<T> v = clear<WHOLE, T>(r[i], col0 + 8 * (id % (2 * CT)), dv, keep_tail || first + row < len);
            if (id < kPieces) __builtin_memcpy(base + row * kRow + 8 * (id % (2 * CT)) * (int)sizeof(T), &v, sizeof(v));
        }
    }
    __device__ __forceinline__ f32x4 get(int j, int n, int p) const {
        f32x4 v;
        if constexpr (sizeof(T) == 2) {
            const vec_t<T, 4> h = __builtin_bit_cast(vec_t<T, 4>, read_tr(base + (4 * p + (n >> 2)) * kRow + 2 * (4 * CT * (n & 3) + 4 * j)));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(h[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const float*>(base + (4 * p + e) * kRow + 4 * col_of<CT>(j, n));
        }
        return v;
    }
};
// A wave's gates: gam, bet, del of its 16 tokens and gam of the chunk's last one, one load for all, through LDS
struct GateTile {
    static constexpr int kBytes = 256;   // per wave
    float* base;
    float r;
    __device__ __forceinline__ void fetch(const float* g, int w, int lane) { r = g[lane < 48 ? (lane >> 4) * C + 16 * w + (lane & 15) : C - 1]; }
    __device__ __forceinline__ void hand(int lane) const { base[lane] = r; }
    __device__ __forceinline__ f32x4 four(int which, int p) const { return *reinterpret_cast<const f32x4*>(base + 16 * which + 4 * p); }
    __device__ __forceinline__ float gam(int n) const { return base[n]; }
    __device__ __forceinline__ float last() const { return base[48]; }
};
template <typename T>
__device__ __forceinline__ Frag<Prec<T>::NX> planes_of(const Raw8<T>& r) {
    Frag<Prec<T>::NX> f;
    if constexpr (Prec<T>::NX == 1) {
        __builtin_memcpy(&f.p[0], &r, 16);
    } else {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(r.v[e]);
        split<Prec<T>::NX>(x, f);
    }
    return f;
}

// B operand that copies columns 16 half .. 16 half + 15 of an operand out of a product: D = A I.  Turns an operand
// whose lanes hold a column (4 consecutive rows in a register each) into one whose lanes hold a row: 8-byte stores instead of 2-byte ones.
template <bool PAIRED = true>
__device__ __forceinline__ bf16x8 unit_frag(int half, int n, int p) {
    bf16x8 f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = static_cast<bf16_t>((PAIRED ? 16 * (e >> 2) + 4 * p + (e & 3) : 8 * p + e) == 16 * half + n ? 1.f : 0.f);
    return f;
}

// ---- a (64 tokens x KP) tile of q or k in LDS: NX planes, rows of 2 KP + 32 bytes (the 16 rows a transposing read touches start 8 banks apart)
template <int KP> constexpr int tile_row() { return 2 * KP + 32; }
template <int KP> constexpr int tile_bytes() { return C * tile_row<KP>(); }
template <int KP, int NX>
__device__ __forceinline__ void tile_put(char* tile, int row, int c, const Frag<NX>& f) {   // columns c .. c+7
#pragma unroll
    for (int i = 0; i < NX; ++i) *reinterpret_cast<bf16x8*>(tile + i * tile_bytes<KP>() + row * tile_row<KP>() + 2 * c) = f.p[i];
}
template <int KP, int NX>
__device__ __forceinline__ Frag<NX> tile_rows(const char* tile, int row, int c) {
    Frag<NX> f;
#pragma unroll
    for (int i = 0; i < NX; ++i) f.p[i] = *reinterpret_cast<const bf16x8*>(tile + i * tile_bytes<KP>() + row * tile_row<KP>() + 2 * c);
    return f;
}
// lane: column 16 m + n, tokens of block tb (32) in paired order.  ds_read_b64_tr_b16: lane i of 16 names row i / 4, column group i % 4
template <int KP, int NX>
__device__ __forceinline__ Frag<NX> tile_cols(const char* tile, int m, int tb, int n, int p) {
    Frag<NX> f;
    const char* at = tile + (32 * tb + 4 * p + (n >> 2)) * tile_row<KP>() + 2 * (16 * m + 4 * (n & 3));
#pragma unroll
    for (int i = 0; i < NX; ++i)
        f.p[i] = join(read_tr(at + i * tile_bytes<KP>()), read_tr(at + i * tile_bytes<KP>() + 16 * tile_row<KP>()));
    return f;
}

// ---- what the waves of a walk hand each other: N planes of a matrix by columns, CT x 16 columns (lane n) x `len` rows of the matrix, 4 consecutive
// ones (a register quadruple) written at a time, 8 (an operand) read.  Rows of 2 len + 16 bytes: 16 lanes of a quarter fall on all banks.
template <int N, int CT, int LEN>
struct Exchange {
    static constexpr int kRow = 2 * LEN + 16, kPlane = CT * 16 * kRow, kBytes = N * kPlane;
    char* base;
    __device__ __forceinline__ void put(int j, int n, int at, const f32x4& v) const {
        float x[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            vec_t<unsigned, 2> u;
            u[0] = take_bf16(x[0], x[1], i + 1 == N);
            u[1] = take_bf16(x[2], x[3], i + 1 == N);
            *reinterpret_cast<vec_t<unsigned, 2>*>(base + i * kPlane + (16 * j + n) * kRow + 2 * at) = u;
        }
    }
    template <int M = N>   // the first M planes
    __device__ __forceinline__ Frag<M> get(int j, int n, int at) const {
        Frag<M> f;
#pragma unroll
        for (int i = 0; i < M; ++i) f.p[i] = *reinterpret_cast<const bf16x8*>(base + i * kPlane + (16 * j + n) * kRow + 2 * at);
        return f;
    }
};
__device__ __forceinline__ int paired(int tile, int p) { return 32 * (tile >> 1) + 8 * p + 4 * (tile & 1); }   // where rows 16 tile + 4 p .. + 3 stand

// ---- lower triangular 64 x 64 matrices (T, M): the six 16 x 32 operands that hold something, in operand order (1 KB each, lane by lane)
constexpr int kTri = 6 * 1024;   // bytes of one plane
__device__ __host__ constexpr int tri(int rt, int kb) { return rt < 2 ? rt : 2 + 2 * (rt - 2) + kb; }
template <int N>
__device__ __forceinline__ Frag<N> tri_rows(const char* m, int rt, int kb, int lane) {   // lane: row 16 rt + n, columns of block kb
    Frag<N> f;
#pragma unroll
    for (int i = 0; i < N; ++i) f.p[i] = *reinterpret_cast<const bf16x8*>(m + i * kTri + 1024 * tri(rt, kb) + 16 * lane);
    return f;
}
// their transposes, for the backward: lane = column 16 ct + n, rows of block ib (those with ib >= ct / 2)
__device__ __host__ constexpr int tri_t(int ct, int ib) { return ct < 2 ? 2 * ct + ib : 4 + (ct - 2); }
template <int N>
__device__ __forceinline__ Frag<N> tri_cols(const char* m, int ct, int ib, int lane) {
    Frag<N> f;
#pragma unroll
    for (int i = 0; i < N; ++i) f.p[i] = *reinterpret_cast<const bf16x8*>(m + i * kTri + 1024 * tri_t(ct, ib) + 16 * lane);
    return f;
}

// L of a pair from the difference of its sums (exponents of 2, at most 0 where the pair counts): the choice is made in the exponent, as a branch around the
// exponential and the reads of its operand costs a latency per element
using f64x4 = vec_t<double, 4>;
__device__ __forceinline__ float decay(bool counts, double d) { return fast_exp2((float)(counts ? d : -1e4)); }

// ---- what a chunk leaves in the workspace; slot = (batch entry * heads + head) * chunks + chunk
struct Gates { float gam[C], bet[C], del[C]; double G[C]; };   // G: the sums of g in units of log 2
struct Layout {
    int64_t tri, gates, S0, U;                      // byte offsets of the arrays in the forward's workspace
    int64_t dS, Y;                                  // ... in the backward's own
    int64_t tri_slot, s_slot, u_slot;               // bytes per chunk (T and M; S0 / dS; U / Y)
    int64_t bytes, bwd_bytes;
    int chunks, vpad;
};
__host__ __device__ __forceinline__ int ceil_to(int a, int b) { return (a + b - 1) / b * b; }
__host__ __device__ __forceinline__ int pad_k(int dk) { return dk <= 64 ? 64 : 128; }
// NB: the planes of what the backward computes and is handed
inline int planes_kept(const vms_gated_delta_params& p) { return p.dtype == VMS_F32 || p.fp32_states ? 3 : 2; }
__host__ inline Layout layout(const vms_gated_delta_params& p) {
    Layout l{};
    const int no = p.dtype == VMS_F32 ? 3 : 2, nb = p.for_backward ? planes_kept(p) : 0;   // Prec<T>::NO, the kernels' NB
    l.chunks = (p.seqlen + C - 1) / C;
    l.vpad = ceil_to(p.dv, 32);
    const int64_t slots = (int64_t)p.batch * p.heads * l.chunks;
    l.tri_slot = (int64_t)(NS + no + 2 * nb) * kTri;   // planes of T, M and, for the backward, their transposes
    l.s_slot = (int64_t)nb * pad_k(p.dk) * l.vpad * 2;
    l.u_slot = (int64_t)nb * C * l.vpad * 2;
    int64_t at = 0;
    auto take = [&](int64_t n) { int64_t o = at; at += (n + 255) / 256 * 256; return o; };
    l.tri = take(slots * l.tri_slot);
    l.gates = take(slots * (int64_t)sizeof(Gates));
    if (p.for_backward) {
        l.S0 = take(slots * l.s_slot);
        l.U = take(slots * l.u_slot);
    }
    l.bytes = at;
    at = 0;
    l.dS = take(slots * l.s_slot);
    l.Y = take(slots * l.u_slot);
    l.bwd_bytes = at;
    return l;
}

// position in memory of the i-th token of the walk (valid for i < len); rows >= len are padding and stay where they are
__device__ __forceinline__ int token(int i, int len, int reverse) { return reverse ? len - 1 - i : i; }
__device__ __forceinline__ int length_of(const vms_gated_delta_params& p, int b) {
    if (!p.seq_lens) return p.seqlen;
    const int n = p.seq_lens[b];
    return n < 0 ? 0 : n > p.seqlen ? p.seqlen : n;
}
// workgroup -> (batch * heads + head, slice): the slices of one head share q, k, T and M, so they go to one XCD's L2 (workgroups
// are dealt to the 8 XCDs in turn)
__device__ __forceinline__ void pair_of(int id, int pairs, int slices, int& pair, int& slice) {
    if (pairs % 8 == 0) {
        const int in = id >> 3;
        slice = in % slices;
        pair = (in / slices) * 8 + (id & 7);
    } else {
        slice = id % slices;
        pair = id / slices;
    }
}

__device__ __forceinline__ float ld_gate(const void* p, int64_t i, int dt) {
    if (dt == VMS_F32) return static_cast<const float*>(p)[i];
    if (dt == VMS_F16) return static_cast<float>(static_cast<const f16_t*>(p)[i]);
    return static_cast<float>(static_cast<const bf16_t*>(p)[i]);
}
inline int allow_lds(PerDeviceOnce& once, const void* kernel, int bytes) {
    if (bytes <= 65536) return VMS_OK;
    const hipError_t e = once.run([&] { return hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes); });
    if (e != hipSuccess) { set_error("hipFuncSetAttribute: %s", hipGetErrorString(e)); return VMS_ERR_LAUNCH; }
    return VMS_OK;
}
// CT accumulator tiles (rows row0 + 4 p + r, column col0 + col_of(j, n)) into N planes of (rows, vpad): through unit_frag, so that a lane
// stores 4 CT consecutive columns of one row.  vpad is a multiple of 32, so that the 16 CT columns of a slice are always inside
template <int N, int CT>
__device__ __forceinline__ void store_rows(char* base, int rows, int vpad, int row0, int col0, const f32x4 (&v)[CT], int n, int p) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    Frag<N> f[CT];
#pragma unroll
    for (int j = 0; j < CT; ++j) f[j] = frag_of<N>(v[j], zero);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        vec_t<bf16_t, 4 * CT> o;
#pragma unroll
        for (int j = 0; j < CT; ++j) {
            const f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[j].p[i], unit_frag(0, n, p), zero, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * j + e] = static_cast<bf16_t>(x[e]);
        }
        *reinterpret_cast<vec_t<bf16_t, 4 * CT>*>(base + 2 * (((int64_t)i * rows + row0 + n) * vpad + col0 + 4 * CT * p)) = o;
    }
}
// The same from operands (lane: column col_of(j, n), 32 rows): rows row0 .. of N planes.  PAIRED: the 16 rows of one half, else both halves
template <int N, int CT, bool PAIRED>
__device__ __forceinline__ void store_frag(char* base, int rows, int vpad, int row0, int half, int col0, const Frag<N> (&f)[CT], int n, int p) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int hh = 0; hh < (PAIRED ? 1 : 2); ++hh) {
            vec_t<bf16_t, 4 * CT> o;
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                const f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[j].p[i], unit_frag<PAIRED>(PAIRED ? half : hh, n, p), zero, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[4 * j + e] = static_cast<bf16_t>(x[e]);
            }
            *reinterpret_cast<vec_t<bf16_t, 4 * CT>*>(base + 2 * (((int64_t)i * rows + row0 + 16 * hh + n) * vpad + col0 + 4 * CT * p)) = o;
        }
}

// A wave's 16 tokens x 16 CT columns of an output, from accumulators [column 4 p + r of tile j][token n] through LDS (a VTile's place) to whole lines
template <typename T, int CT, bool WHOLE>
struct OTile {
    char* base;
    static constexpr int kRow = VTile<T, CT, WHOLE>::kRow;
    __device__ __forceinline__ void put(const f32x4 (&v)[CT], int lane) const {
        vec_t<T, 4 * CT> o;
#pragma unroll
        for (int e = 0; e < 4 * CT; ++e) o[e] = static_cast<T>(v[e >> 2][e & 3]);
        __builtin_memcpy(__builtin_assume_aligned(base + (lane & 15) * kRow + 4 * CT * (lane >> 4) * (int)sizeof(T), 8), &o, sizeof(o));
    }
    __device__ __forceinline__ void store(const Rows<T>& out, int first, int len, int col0, int dv, int lane) const {
        const int id = lane & (32 * CT - 1), row = id / (2 * CT), c = col0 + 8 * (id % (2 * CT));
        Raw8<T> r;
        __builtin_memcpy(&r, __builtin_assume_aligned(base + row * kRow + 8 * (id % (2 * CT)) * (int)sizeof(T), 16), sizeof(r));
        if (lane < 32 * CT && first + row < len) {
            T* const at = const_cast<T*>(out.row(first + row)) + c;
            if (WHOLE) {
                if (c < dv) __builtin_memcpy(at, &r, sizeof(r));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < dv) at[e] = r.v[e];
            }
        }
    }
};

// A walk's workgroup takes 32 columns of a head, or 16 where that leaves half of the CUs without one: a chunk of 16 columns takes 0.65 .. 0.75 of the time of one of
// 32 (its chain is the same).  Forward / backward walk, us, 32 against 16 columns (bf16):
//   (2, 2304, 8 heads, 64 x 64)      32 workgroups 77 / 72      64 workgroups 56 / 50
//   (8, 3136, 6 heads, 128 x 128)   192 workgroups 184 / 168   384 workgroups 267 / 264
//   (8, 8192, 8 heads, 128 x 128)   256 workgroups 388         512 workgroups 492
inline bool narrow(const vms_gated_delta_params& p, const Layout& l) { return (int64_t)p.batch * p.heads * (l.vpad / 32) <= device_cu_count() / 2; }

// The most columns that the backward's walk takes: the planes of fp32, and three of fp16 beside 128-wide keys, leave LDS for one column tile
constexpr int bwd_columns(int dtype, int planes, int kp) { return dtype == VMS_F32 || (dtype == VMS_F16 && planes == 3 && kp == 128) ? 16 : 32; }

int validate(const vms_gated_delta_params& p);   // gated_delta_fwd.hip

}  // namespace gd
}  // namespace vms
