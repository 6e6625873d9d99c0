// attn_kernels.hip -- attention over a paged cache and over packed prompts, the
// cache's copies, rows on their way into and out of it, and the selection of beams
// (sllm_gfx950_attn.h), for gfx950.
//
// Attention of a row: out = sum_j p_j v_j / sum_j p_j, p_j = 2^(c (s_j - m)),
// s_j = q . k_j, c = scale log2(e), m a running maximum of s. One pass over the
// keys: m, the sum l and the sums of p v are carried in f32 registers and scaled
// down when a larger s comes.
//
// A row is a query token and one of the query heads of a KV head, so that the
// heads that share keys share the tile that holds them. The scores are formed
// as S^T = K Q^T with 16 x 16 matrix instructions: a lane then holds scores of
// one row (lane % 16) for four keys (4 (lane / 16) + i), which is the operand
// layout that O^T += V^T P^T wants, so p never leaves its lane; only a tile's
// maximum crosses lanes.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_layout.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Pointers read from memory or built from integers are generic to the compiler
// and would be accessed with flat instructions, which count against the LDS
// counter too: these name the address space.
#define GLOBAL __attribute__((address_space(1)))
#define G_CAST(T, p) ((GLOBAL T *) (p))
// Tables that no kernel writes: with an address that is the same for the whole
// wave these are scalar loads, which do not queue behind the tiles' copies.
#define C_CAST(T, p) ((__attribute__((address_space(4))) const T *) (p))
#define LDS_PTR(p) ((__attribute__((address_space(3))) void *) (p))

constexpr int WAVES = 4;

// what copies to LDS read in place of keys past the end and dimensions past head_dim
__device__ __attribute__((aligned(16))) uint32_t att_zeros[4];

template <int N> __device__ __forceinline__ void wait_vmem() {   // s_waitcnt vmcnt(N), the other counters untouched
    static_assert(N >= 0 && N < 64, "vmcnt");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t) __builtin_amdgcn_readfirstlane((int) x); }

// over the four lanes that hold a row (lane, lane ^ 16, lane ^ 32, lane ^ 48)
__device__ __forceinline__ float row_max(float x) {
    u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_sum(float x) {
    u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <typename T> struct vec8 { typedef T type __attribute__((ext_vector_type(8))); };
template <typename T> struct is_f16 { static constexpr bool value = false; };
template <> struct is_f16<_Float16> { static constexpr bool value = true; };
template <typename X, typename Y> struct is_same { static constexpr bool value = false; };
template <typename X> struct is_same<X, X> { static constexpr bool value = true; };
template <typename T> struct vec4 { typedef T type __attribute__((ext_vector_type(4))); };

__device__ __forceinline__ f32x4 mfma(vec8<_Float16>::type a, vec8<_Float16>::type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(vec8<__bf16>::type a, vec8<__bf16>::type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// a + b + c, the first two exactly (f16's subnormals too)
__device__ __forceinline__ float add_two(_Float16 a, _Float16 b, float c) {
    typedef _Float16 two __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2((two) { a, b }, (two) { (_Float16) 1.0f, (_Float16) 1.0f }, c, false);
}
__device__ __forceinline__ float add_two(__bf16 a, __bf16 b, float c) {
    typedef __bf16 two __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16((two) { a, b }, (two) { (__bf16) 1.0f, (__bf16) 1.0f }, c, false);
}

constexpr float LOWEST = -3.402823466e38f;

// what a cache of 8 bits holds
struct int8_codes {};
struct e4m3_codes {};

// Codes and their scale as bf16, which holds each of their products exactly (S is 0 where
// the byte is, of rows that are not there, whose codes are 0).
__device__ __forceinline__ float scale_value(uint32_t byte) { return __uint_as_float(byte << 23); }
template <typename S> __device__ __forceinline__ u32x2 values_of_codes(uint32_t v, float by) {
    typedef __bf16 two __attribute__((ext_vector_type(2)));
    two a, b;
    if constexpr (is_same<S, int8_codes>::value) {
        const uint32_t u = v ^ 0x80808080u;                      // code + 128
        const float off = -128.0f * by;
        a = (two) { (__bf16) fmaf((float) (u & 255u), by, off), (__bf16) fmaf((float) (u >> 8 & 255u), by, off) };
        b = (two) { (__bf16) fmaf((float) (u >> 16 & 255u), by, off), (__bf16) fmaf((float) (u >> 24), by, off) };
    } else {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, by, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, by, true);
    }
    return (u32x2) { __builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b) };
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------

// Keys of a tile and what it takes in LDS: its keys' rows of D values, then its
// values' rows, 16-byte pieces of a row swapped about by the row (ksw, vsw) so
// that the lanes of one read fall into different banks. KEYS: a wave's own tiles,
// whose keys go to registers, so that a stage is its values alone.
template <typename T, int D, bool KEYS> struct tile {
    static constexpr bool WIDE = sizeof(T) == 4;
    static constexpr int KT = WIDE ? 16 : 32;
    static constexpr int ROWB = D * (int) sizeof(T);
    static constexpr int CH = ROWB / 16;
    static constexpr int HALF = KT * ROWB;
    static constexpr int VALUES = KEYS ? 0 : HALF;               // where the values are
    static constexpr int BYTES = VALUES + HALF;
    static constexpr int STAGES = KEYS ? 1 : 4;
    static constexpr int LDS = BYTES * STAGES * (KEYS ? WAVES : 1);
    static __device__ __forceinline__ uint32_t ksw(uint32_t r) { return !WIDE && CH == 16 ? r & 15u : r & 7u; }
    static __device__ __forceinline__ uint32_t vsw(uint32_t r) {
        if (WIDE) return (CH == 32 ? (r >> 2) & 7u : (r >> 2) & 3u) << 2;
        return (CH == 16 ? r & 7u : (r >> 1) & 3u) << 1;
    }
};

// A: the type of q and out. T: of the keys and values. D: head_dim, padded. A
// wave has NT tiles of 16 rows. KEYS: the waves take the item's tiles in turn,
// all for the same rows, and their results are joined in LDS; else each wave
// has rows of its own and all share a tile. PAGED: keys are found by page. C: what a
// cache of 8 bits holds, T what its values are turned into on their way to LDS or to the
// products: bf16, which holds a code times its scale exactly. Queries are then sums of bf16
// values, one for rows of bf16, two for f16 (all 11 bits), three for f32 (24), and weights
// likewise; but of rows of bf16 with up to 64 a workgroup they are sums of two, 16 bits, which
// leaves a result's own rounding (1.67e-3 of it on average; with 8 bits of a weight 2.0e-3 to 2.2e-3).
// That costs nothing where memory bounds (8 sequences of up to 65536 positions 57.4 and
// 57.5 us) and 4 to 7 % behind shared prefixes (64 sequences behind 4096 positions 24.6 and 25.7,
// drafts of 5 27.0 and 28.8), but 22 % in 128 rows, which the products bound (4 times
// 512 new positions 83.9 and 102.7 us): there weights have the 8 bits of the rows' type.
template <typename A, typename T, int D, int NT, bool KEYS, bool PAGED, typename C = T>
struct attention {
    typedef tile<T, D, KEYS> L;
    static constexpr bool WIDE = L::WIDE;
    static constexpr bool HELD8 = !is_same<C, T>::value;
    static constexpr bool SPLIT = !HELD8 && !WIDE && sizeof(A) == 4;       // f32 rows against f16 keys
    static constexpr int PIECES = !HELD8 ? 1 : sizeof(A) == 4 ? 3 : is_f16<A>::value ? 2 : 1;
    static constexpr int WEIGHT = HELD8 && PIECES == 1 && NT == 1 ? 2 : PIECES;
    // values beside the first that a query, and that a weight is the sum of
    static constexpr int MORE = PIECES - 1 + SPLIT, MOREW = WEIGHT - 1 + SPLIT;
    static constexpr int KT = L::KT;
    static constexpr int KS = KT / 16;                           // 16-key subtiles
    static constexpr int DT = D / 16;
    static constexpr int QC = D * (int) sizeof(T) / 64;          // 16-byte pieces of a row that a lane holds
    static constexpr int GROUP = KEYS ? 16 : KT / WAVES;   // rows that one address serves: within a page
    static constexpr int GROUPS = (KEYS ? KT : KT / WAVES) / GROUP;
    static constexpr int RPI = 1024 / L::ROWB;                   // rows of a copy instruction
    typedef typename vec8<T>::type t8;

    static constexpr int COPIES = GROUP / RPI;                   // instructions of a group, for keys and for values
    static constexpr uint32_t PAST = 0xfffffff0u;                // a place past any end
    static constexpr int DA = WIDE ? 4 : 2;                      // 16-byte pieces of 16 dimensions
    static constexpr int VM = 2 * COPIES;                        // a wave's copies for a tile (not KEYS)
    // 8 bits: 16-byte pieces of codes. A lane's of a row of keys (KEYS), lanes a row of
    // values (not KEYS: of either), and instructions of a group's
    static constexpr int KL = D / 64, LPR = D / 16, CL = GROUP * LPR > 64 ? GROUP * LPR / 64 : 1;

    const att_args &a;
    const att_item it;
    uint8_t *S;
    uint32_t lane, wave, g, li;

    // What a lane adds to a tile's place in LDS, once for all tiles. Keys: row li of a
    // 16-key subtile, piece 4 q + g; the row's swap is the same in every subtile.
    // Values: dimension tile 0 of row 4 g (16 bits: 4 g + li / 4, of the transposing
    // read; f32: 4 g + i, a row further each); dimension tile dt is at ^ dt * 16 DA.
    uint32_t koff[QC], voff;
    // a lane's place in the rows that a copy instruction fills, or past any end where
    // the row has no such piece
    // KEYS: keys are read as the products take them, and values are swapped when they
    // are written to LDS, at vput.
    uint32_t kcopy[KEYS ? QC : COPIES], vcopy[COPIES], vput[KEYS ? COPIES : 1];
    // 8 bits: kcopy and vcopy are places of codes, krow and vrow of their scales; where a
    // row's two pieces of T go in LDS
    uint32_t krow, vrow[HELD8 ? CL : 1], kput2[2], vput2[HELD8 ? CL : 1][2];

    // the first of the eight dimensions that a lane's step q of the products takes (any
    // order does if queries and keys have the same)
    __device__ __forceinline__ uint32_t dim(int q) const {
        return HELD8 && KEYS ? 64u * (q >> 1) + 16u * g + 8u * (q & 1) : 8u * (4u * q + g);
    }

    __device__ __forceinline__ void places8() {
        const uint32_t ch = lane % LPR;
        krow = KEYS ? li : lane / LPR < (uint32_t) GROUP ? lane / LPR : PAST;
#pragma unroll
        for (int j = 0; j < KL && KEYS; ++j) kcopy[j] = (4u * j + g) * 16u < a.hd ? li * a.hd + (4u * j + g) * 16u : PAST;
        if (!KEYS) kcopy[0] = ch * 16u < a.hd && krow != PAST ? krow * a.hd + ch * 16u : PAST;
#pragma unroll
        for (int j = 0; j < CL; ++j) {
            const uint32_t rg = (uint32_t) j * (64 / LPR) + lane / LPR;
            vrow[j] = rg < (uint32_t) GROUP ? rg : PAST;
            vcopy[j] = ch * 16u < a.hd && vrow[j] != PAST ? rg * a.hd + ch * 16u : PAST;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t rt = KEYS ? rg : wave * (uint32_t) GROUP + rg;
                vput2[j][e] = L::VALUES + rt * L::ROWB + ((2u * ch + e) ^ L::vsw(rt)) * 16u;
                if (!KEYS) kput2[e] = rt * L::ROWB + ((2u * ch + e) ^ L::ksw(rt)) * 16u;
            }
        }
    }

    __device__ __forceinline__ void places() {
        if constexpr (HELD8) places8();
        const uint32_t row = a.hd * (uint32_t) sizeof(T);
        const uint32_t rowk = PAGED ? row : (uint32_t) a.k_tok, rowv = PAGED ? row : (uint32_t) a.v_tok;
#pragma unroll
        for (int q = 0; q < QC; ++q) {
            if (!KEYS) koff[q] = li * L::ROWB + (((4u * q + g) ^ L::ksw(li)) * 16u);
            else if (!HELD8) kcopy[q] = (4u * q + g) * 16u < row ? li * rowk + (4u * q + g) * 16u : PAST;
        }
        const uint32_t r = WIDE ? 4u * g : 4u * g + (li >> 2);
        voff = L::VALUES + r * L::ROWB + (WIDE ? ((li >> 2) ^ L::vsw(r)) * 16u + (li & 3u) * 4u
                                             : (((li >> 1) & 1u) ^ L::vsw(r)) * 16u + (li & 1u) * 8u);
#pragma unroll
        for (int j = 0; j < COPIES && !HELD8; ++j) {
            const uint32_t rg = (uint32_t) j * RPI + lane / L::CH, ch = lane % L::CH;
            if constexpr (KEYS) {                                // (16 rows further on: the same swap)
                vcopy[j] = ch * 16u < row ? rg * rowv + ch * 16u : PAST;
                vput[j] = rg * L::ROWB + (ch ^ L::vsw(rg)) * 16u;
                continue;
            }
            const uint32_t rt = wave * (uint32_t) GROUP + rg;
            const uint32_t ck = (ch ^ L::ksw(rt)) * 16u, cv = (ch ^ L::vsw(rt)) * 16u;
            kcopy[j] = ck < row ? rg * rowk + ck : PAST;
            vcopy[j] = cv < row ? rg * rowv + cv : PAST;
        }
    }

    // rows: lane li of row tile nt
    int lim[NT];                    // keys the row sees
    float c[NT];
    float m[NT], l[NT];             // c times the running maximum (- UP), and the lane's share of the sum
    f32x4 o[DT][NT];
    // a lane's pieces of q: 8 values (SPLIT: and what rounding left of them), or 4 f32
    t8 qf[WIDE ? 1 : NT][WIDE ? 1 : QC], ql[MORE ? NT : 1][MORE ? QC : 1], qm[MORE > 1 ? NT : 1][MORE > 1 ? QC : 1];
    f32x4 qw[WIDE ? NT : 1][WIDE ? QC : 1];
    int lim_min;                    // of the wave's rows

    __device__ __forceinline__ uint32_t row_of(int nt) const {
        return min((KEYS ? 0u : wave * (16u * NT)) + 16u * (uint32_t) nt + li, it.n_rows - 1u);
    }
    // the token and the head of one of the item's rows (h0 + row is small: the product
    // with 1 / group, half a step up, is rounded down to the quotient without error)
    struct place { uint32_t t, h; };
    __device__ __forceinline__ place place_of(uint32_t row) const {
        const uint32_t x = it.h0 + row, t = (uint32_t) (((float) x + 0.5f) * a.per_group);
        return { it.t0 + t, it.head * a.group + x - t * a.group };
    }
    __device__ __forceinline__ uint32_t token(uint32_t t) const {
        return it.list == ATT_TOKENS ? it.tok0 + t : *G_CAST(const uint32_t, a.list + it.list + t);
    }
    __device__ __forceinline__ int limit(uint32_t t) const {     // (vis0 + t, at most the range's end)
        return min((int) it.key1, it.vis0 + (int) t);
    }

    // x as a sum of N (2, 3) bf16 values: cut off, so that none is over x where x is near f32's
    // end, and what is left rounded to the last
    template <int N> __device__ __forceinline__ static void pieces(float x, T (&p)[3]) {
        const float hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
        p[0] = (T) hi;
        x -= hi;
        if constexpr (N > 2) {
            const float mid = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
            p[1] = (T) mid;
            p[2] = (T) (x - mid);
        } else {
            p[1] = (T) x;
        }
    }

    __device__ __forceinline__ void load_q() {
        const uint32_t first = KEYS ? 0u : wave * (16u * NT);
        lim_min = limit(place_of(min(first, it.n_rows - 1u)).t);
        lim_min = (int) uniform((uint32_t) lim_min);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const place at = place_of(row_of(nt));
            lim[nt] = limit(at.t);
            const uint8_t *src = (const uint8_t *) a.q + token(at.t) * a.q_tok + at.h * a.q_head;
            c[nt] = a.c;
            if constexpr (WIDE) {
#pragma unroll
                for (int s = 0; s < QC; ++s) {
                    const uint32_t d = 4u * (4u * s + g);
                    qw[nt][s] = d < a.hd ? *G_CAST(const f32x4, src + d * 4u) : (f32x4) { 0, 0, 0, 0 };
                }
            } else if constexpr (PIECES > 1) {
#pragma unroll
                for (int s = 0; s < QC; ++s) {
                    const uint32_t d = dim(s);
                    float x[8];
                    if constexpr (sizeof(A) == 4) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const f32x4 v = d < a.hd ? *G_CAST(const f32x4, src + d * 4u + 16u * i) : (f32x4) { 0, 0, 0, 0 };
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[4 * i + e] = v[e];
                        }
                    } else {
                        const u32x4 v = d < a.hd ? *G_CAST(const u32x4, src + d * 2u) : (u32x4) { 0, 0, 0, 0 };
                        const typename vec8<A>::type y = __builtin_bit_cast(typename vec8<A>::type, v);
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = (float) y[e];
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        T p[3];
                        pieces<PIECES>(x[e], p);
                        qf[nt][s][e] = p[0];
                        ql[nt][s][e] = p[1];
                        if constexpr (PIECES > 2) qm[nt][s][e] = p[2];
                    }
                }
            } else if constexpr (!SPLIT) {
#pragma unroll
                for (int s = 0; s < QC; ++s) {
                    const uint32_t d = dim(s);
                    const u32x4 v = d < a.hd ? *G_CAST(const u32x4, src + d * 2u) : (u32x4) { 0, 0, 0, 0 };
                    qf[nt][s] = __builtin_bit_cast(t8, v);
                }
            } else {
                // f32 queries as the sum of two f16 values. The row is first scaled by a
                // power of two to a largest magnitude of 2^14..2^15, the upper end of f16's
                // range; c takes the power back. So an element keeps 22 bits down to 2^-17 of
                // the largest, and below that is off by at most 2^-39 of it (at 1..2 it was
                // 2^-25, which a key's large element makes a score's largest error).
                f32x4 x[QC][2];
                float top = 0.0f, least = -LOWEST;
#pragma unroll
                for (int s = 0; s < QC; ++s) {
                    const uint32_t d = 8u * (4u * s + g);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        x[s][i] = d < a.hd ? *G_CAST(const f32x4, src + d * 4u + 16u * i) : (f32x4) { 0, 0, 0, 0 };
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            top = fmaxf(top, fabsf(x[s][i][e]));
                            least = fminf(least, d < a.hd ? fabsf(x[s][i][e]) : -LOWEST);
                        }
                    }
                }
                top = row_max(top);
                const int up = 15 - __builtin_amdgcn_frexp_expf(top);        // (the exponent of 0 is 0)
                // not 0, which times a masked -inf is NaN, nor infinite: scores this small or
                // large make the weights 1, or 0 and 1, whatever c is exactly
                c[nt] = fminf(fmaxf(__builtin_amdgcn_ldexpf(a.c, -up), 0x1p-126f), -LOWEST);
#pragma unroll
                for (int s = 0; s < QC; ++s) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float f = __builtin_amdgcn_ldexpf(x[s][e >> 2][e & 3], up);
                        const T hi = (T) f;
                        qf[nt][s][e] = hi;
                        ql[nt][s][e] = (T) (f - (float) hi);
                    }
                }
                // An element too small for f16 keeps its sign, as f16's smallest, for infinite
                // elements of keys; what is left of it is the difference. (Such rows alone: for
                // every row it is 0.6 us of a step of 64 sequences behind 4096 positions.)
                if (__any(__builtin_amdgcn_ldexpf(least, up) < 0x1p-24f)) {
#pragma unroll
                    for (int s = 0; s < QC; ++s) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float f = __builtin_amdgcn_ldexpf(x[s][e >> 2][e & 3], up);
                            if (f == 0.0f || qf[nt][s][e] != (T) 0.0f) continue;
                            qf[nt][s][e] = (T) copysignf(0x1p-24f, f);
                            ql[nt][s][e] = (T) (f - copysignf(0x1p-24f, f));
                        }
                    }
                }
            }
        }
    }

    // Where GROUP rows of keys and of values are, from `key` on (of which the rows below
    // the range's end are read).
    // (8 bits: off is where a block's codes and scales are, and `slot` the first row.)
    struct span { const uint8_t *k, *v; uint32_t slot; };
    __device__ __forceinline__ span rows_at(uint32_t key) const {
        if constexpr (HELD8) {
            const uint32_t at = min(key, it.key1 - 1u);
            const uint32_t page = *C_CAST(uint32_t, a.tables + it.kv + (at >> a.page_shift));
            const uint64_t off = page * a.page_bytes + (uint64_t) it.head * a.block_bytes;
            return { a.k + off, a.v + off, at & ((1u << a.page_shift) - 1u) & ~(uint32_t) (GROUP - 1) };
        } else if constexpr (PAGED) {
            const uint32_t at = min(key, it.key1 - 1u);
            const uint32_t page = *C_CAST(uint32_t, a.tables + it.kv + (at >> a.page_shift));
            const uint64_t off = page * a.page_bytes + ((uint64_t) (it.head << a.page_shift) + (at & ((1u << a.page_shift) - 1u) & ~(uint32_t) (GROUP - 1))) * (a.hd * (uint32_t) sizeof(T));
            return { a.k + off, a.v + off, 0 };
        } else {
            return { a.k + (uint64_t) (it.kv + key) * a.k_tok + it.head * a.k_head, a.v + (uint64_t) (it.kv + key) * a.v_tok + it.head * a.v_head, 0 };
        }
    }

    // Copy rows straight to LDS at `to`. `whole`: all of them, of full length, are there;
    // else those from `n` on and what is past head_dim arrive as zeros.
    __device__ __forceinline__ void copy_rows(const uint8_t *from, const uint32_t (&place)[COPIES], uint32_t to, bool whole, uint32_t n) const {
        if (whole) {
#pragma unroll
            for (int j = 0; j < COPIES; ++j) __builtin_amdgcn_global_load_lds((const void *) (from + place[j]), LDS_PTR(S + to + j * 1024), 16, 0, 0);
        } else {
#pragma unroll
            for (int j = 0; j < COPIES; ++j) {
                const bool in = (uint32_t) j * RPI + lane / L::CH < n && place[j] != PAST;
                __builtin_amdgcn_global_load_lds((const void *) (in ? from + place[j] : (const uint8_t *) att_zeros), LDS_PTR(S + to + j * 1024), 16, 0, 0);
            }
        }
    }
    // rows of a group of tile row r0 that are below the range's end, and whether a tile's all are
    __device__ __forceinline__ uint32_t rows_in(uint32_t key) const { return key < it.key1 ? min(it.key1 - key, (uint32_t) GROUP) : 0u; }
    __device__ __forceinline__ bool is_whole(uint32_t t) const { return (t + 1u) * KT <= it.key1 && a.hd == D; }

    // 8 bits: a group's codes and scales on their way in registers (by a buffer's bounds, what
    // is past the end or past head_dim is zero)
    struct codes {
        u32x4 k[KEYS ? KL : 1], v[CL];
        uint32_t ks, vs[CL];
    };
    // a sequence's own keys are read once and not kept (2: nontemporal): 64.9 -> 60.6 us
    // for 8 sequences of 16384 positions, bf16; a prompt's are read by many workgroups
    static constexpr int KEPT = PAGED ? 2 : 0;
    __device__ __forceinline__ void fetch8(codes &x, const span &m, uint32_t key) const {
        const uint32_t n = rows_in(key);
        const uint8_t *k = m.k + m.slot * a.hd, *v = m.v + m.slot * a.hd;
        const uint32_t scales = (a.hd << a.page_shift) + m.slot;
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void *) k, (short) 0, (int) uniform(n * a.hd), 0x00020000);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void *) v, (short) 0, (int) uniform(n * a.hd), 0x00020000);
        const __amdgpu_buffer_rsrc_t sk = __builtin_amdgcn_make_buffer_rsrc((void *) (m.k + scales), (short) 0, (int) uniform(n), 0x00020000);
        const __amdgpu_buffer_rsrc_t sv = __builtin_amdgcn_make_buffer_rsrc((void *) (m.v + scales), (short) 0, (int) uniform(n), 0x00020000);
        constexpr int KEEP = KEYS ? KEPT : 0;                    // (of scales a line is of several tiles: kept, 59.4 -> 58.0 us)
#pragma unroll
        for (int j = 0; j < (KEYS ? KL : 1); ++j) x.k[j] = __builtin_amdgcn_raw_buffer_load_b128(rk, kcopy[j], 0, KEEP);
        x.ks = __builtin_amdgcn_raw_buffer_load_b8(sk, krow, 0, 0);
#pragma unroll
        for (int j = 0; j < CL; ++j) {
            x.v[j] = __builtin_amdgcn_raw_buffer_load_b128(rv, vcopy[j], 0, KEEP);
            x.vs[j] = __builtin_amdgcn_raw_buffer_load_b8(sv, vrow[j], 0, 0);
        }
    }
    // sixteen codes as two pieces of T
    struct two { u32x4 p[2]; };
    __device__ __forceinline__ static two widen(const u32x4 &v, uint32_t scale) {
        const float by = scale_value(scale);
        two y;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const u32x2 lo = values_of_codes<C>(v[2 * e], by), hi = values_of_codes<C>(v[2 * e + 1], by);
            y.p[e] = (u32x4) { lo[0], lo[1], hi[0], hi[1] };
        }
        return y;
    }
    // a group's values (KEYS) or keys and values into LDS, at `to` more than their places
    __device__ __forceinline__ void land(const codes &x, uint32_t to) const {
        if (!KEYS && krow != PAST) {
            const two y = widen(x.k[0], x.ks);
#pragma unroll
            for (int e = 0; e < 2; ++e) *reinterpret_cast<u32x4 *>(S + to + kput2[e]) = y.p[e];
        }
#pragma unroll
        for (int j = 0; j < CL; ++j) {
            if (vrow[j] == PAST) continue;
            const two y = widen(x.v[j], x.vs[j]);
#pragma unroll
            for (int e = 0; e < 2; ++e) *reinterpret_cast<u32x4 *>(S + to + vput2[j][e]) = y.p[e];
        }
    }
    // Tiles whose rows are in registers (not KEYS): two where 128 rows of bf16 leave room for
    // them: 64 sequences behind 16000 shared positions 43.2 -> 41.7 us, 4 times 512 new positions behind 4000
    // 88.4 -> 85.5; with 64 rows, and with f16's or f32's more registers, one was 1 to 3 % faster.
    static constexpr int SETS = NT == 2 && PIECES == 1 ? 2 : 1;
    codes c8[HELD8 ? (KEYS ? GROUPS : SETS) : 1];
    // not KEYS, 8 bits: this wave's rows of a tile set off
    template <int B> __device__ __forceinline__ void issue8(uint32_t t) {
        const uint32_t key = t * KT + wave * (uint32_t) GROUP;
        fetch8(c8[B], rows_at(key), key);
    }

    // not KEYS: this wave's rows of a tile into the stage at `to`
    __device__ __forceinline__ void issue(uint32_t t, uint32_t to) const {
        const uint32_t r0 = wave * (uint32_t) GROUP;             // row in the tile
        const span m = rows_at(t * KT + r0);
        const bool whole = is_whole(t);
        const uint32_t n = rows_in(t * KT + r0);
        copy_rows(m.k, kcopy, to + r0 * L::ROWB, whole, n);
        copy_rows(m.v, vcopy, to + L::VALUES + r0 * L::ROWB, whole, n);
    }
    // KEYS: a tile's keys, as the products take them, and its values, on their way in
    // registers. What is past the end or past head_dim is zero.
    struct load {
        u32x4 k[KEYS ? KS : 1][KEYS ? QC : 1], v[KEYS ? GROUPS : 1][KEYS ? COPIES : 1];
    };
    struct span_of_tile { span m[GROUPS]; };
    __device__ __forceinline__ span_of_tile spans(uint32_t t) const {
        span_of_tile x;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) x.m[gr] = rows_at(t * KT + (uint32_t) gr * GROUP);
        return x;
    }
    __device__ __forceinline__ void fetch(load &x, const span_of_tile &at, uint32_t t) const {
        __amdgpu_buffer_rsrc_t k[GROUPS], v[GROUPS];
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {
            const uint32_t n = rows_in(t * KT + (uint32_t) gr * GROUP), row = a.hd * (uint32_t) sizeof(T);
            const uint32_t rowk = PAGED ? row : (uint32_t) a.k_tok, rowv = PAGED ? row : (uint32_t) a.v_tok;
            k[gr] = __builtin_amdgcn_make_buffer_rsrc((void *) at.m[gr].k, (short) 0, (int) uniform(n ? n * rowk - (rowk - row) : 0u), 0x00020000);
            v[gr] = __builtin_amdgcn_make_buffer_rsrc((void *) at.m[gr].v, (short) 0, (int) uniform(n ? n * rowv - (rowv - row) : 0u), 0x00020000);
        }
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {
#pragma unroll
            for (int q = 0; q < QC; ++q) x.k[gr][q] = __builtin_amdgcn_raw_buffer_load_b128(k[gr], kcopy[q], 0, KEPT);
        }
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {
#pragma unroll
            for (int j = 0; j < COPIES; ++j) x.v[gr][j] = __builtin_amdgcn_raw_buffer_load_b128(v[gr], vcopy[j], 0, KEPT);
        }
    }

    // A value of the tile that is infinite or NaN.
    __device__ __forceinline__ static bool odd(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

    typedef f32x4 scores[KS][NT];

    // CAREFUL, SPLIT: what rounding left of a query may be 0 or of the other sign, and times
    // an infinite element of a key would be NaN where the product is infinite: the rest is
    // multiplied by 0 there.
    template <bool CAREFUL>
    __device__ __forceinline__ void score(f32x4 (&s)[NT], const u32x4 &piece, int q) const {
        if constexpr (WIDE) {
            const f32x4 kf = __builtin_bit_cast(f32x4, piece);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt] = mfma(kf[e], qw[nt][q][e], s[nt]);
            }
        } else {
            const t8 kf = __builtin_bit_cast(t8, piece);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt] = mfma(kf, qf[nt][q], s[nt]);
            if constexpr (PIECES > 1) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt] = mfma(kf, ql[nt][q], s[nt]);
            }
            if constexpr (PIECES > 2) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt] = mfma(kf, qm[nt][q], s[nt]);
            }
            if constexpr (SPLIT) {
                t8 kr = kf;
                if constexpr (CAREFUL) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) kr[e] = odd((float) kr[e]) ? (T) 0.0f : kr[e];
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt] = mfma(kr, ql[nt][q], s[nt]);
            }
        }
    }

    // keys that a row does not see, of the tile from `key` on (a branch around the scores
    // alone: two copies of the products would each keep the sums in registers of their own)
    __device__ __forceinline__ void mask(scores &s, uint32_t key) const {
        if ((int) (key + KT) <= lim_min) return;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[ks][nt][i] = (int) (key + 16u * ks + 4u * g + i) < lim[nt] ? s[ks][nt][i] : -INFINITY;
            }
        }
    }

    // p of a tile as the products take it: the cache's type (SPLIT: and what rounding to
    // it left), or f32. Rounding p to 16 bits halves the products and their operands, and
    // makes a result's error up to 1.4 times what rounding the result alone leaves. The sum is
    // of p as it was rounded, so that weights still add up to 1: values that are all alike
    // come back as they are (they were 0.4 % off where bf16 rounded all weights one way).
    struct probs {
        t8 p[WIDE ? 1 : NT], rest[MOREW ? NT : 1], last[MOREW > 1 ? NT : 1];
        f32x4 w[WIDE ? NT : 1];
    };

    // The maximum moves only where a score is over it by 8 or more (as a power of two):
    // until then weights are at most 256 times what they were when it moved, which costs no
    // precision, the sums need no scaling, and the lanes that hold a row need not agree on its
    // largest score. m is UP below the maximum, so weights are 2^UP where it moved and up to
    // 2^(UP + 8) after. f32 and bf16, whose values may be as large as f32 holds: at most 1, so
    // that sums overflow no sooner than with the true maximum (at 256 they did; values under
    // 2^-118 lose bits to it instead). f16: at most 2^15, which it holds, so that its
    // smallest, 2^-24, is 2^-31 or less of a row's largest weight and not 2^-24 (the share of
    // 4000 keys with weights about 2^-25 of one's was 0.8 % off); its values times that are
    // far from f32's end. The sums and the parts of a split carry the factor alike. Whether
    // any moved; then f is what the sums of products so far are to be scaled by.
    static constexpr float UP = is_f16<T>::value ? 7.0f : -8.0f;
    __device__ __forceinline__ bool adjust(const scores &s, float (&f)[NT]) {
        float top[NT];
        bool over = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            top[nt] = s[0][nt][0];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int i = 0; i < 4; ++i) top[nt] = fmaxf(top[nt], s[ks][nt][i]);
            }
            over |= fmaf(top[nt], c[nt], -m[nt]) > 8.0f + UP;
        }
        if (!__any(over)) return false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float t = row_max(top[nt]), to = fmaf(t, c[nt], -m[nt]) > 8.0f + UP ? t * c[nt] - UP : m[nt];   // (by the row's own scores alone)
            f[nt] = __builtin_amdgcn_exp2f(m[nt] - to);
            l[nt] *= f[nt];
            m[nt] = to;
        }
        return true;
    }
    // s to p (m is at least the lowest float: a masked -inf gives 2^-inf = 0 and never inf - inf)
    __device__ __forceinline__ void soften(const scores &s, probs &p) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float sum = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[ks][nt][i], c[nt], -m[nt]));
                    if constexpr (WIDE || WEIGHT > 1) sum += x;
                    if constexpr (WIDE) {
                        p.w[nt][i] = x;
                    } else if constexpr (WEIGHT > 1) {           // (16 or more bits of x: as good as x in the sum)
                        T y[3];
                        pieces<WEIGHT>(x, y);
                        p.p[nt][4 * ks + i] = y[0];
                        p.rest[nt][4 * ks + i] = y[1];
                        if constexpr (WEIGHT > 2) p.last[nt][4 * ks + i] = y[2];
                    } else {
                        p.p[nt][4 * ks + i] = (T) x;
                        if constexpr (SPLIT) p.rest[nt][4 * ks + i] = (T) (x - (float) p.p[nt][4 * ks + i]);
                    }
                }
            }
            if constexpr (!WIDE && WEIGHT == 1) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    sum = add_two(p.p[nt][e], p.p[nt][e + 1], sum);
                    if constexpr (SPLIT) sum = add_two(p.rest[nt][e], p.rest[nt][e + 1], sum);
                }
            }
            l[nt] += sum;
        }
    }

    __device__ __forceinline__ void rescale(const float (&f)[NT]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt][nt] *= f[nt];
        }
    }

    // A tile's values as the products take them: keys 4 g + 0..3 of each 16-key subtile, by
    // a transposing read (16 bits); one key an instruction (f32: not held).
    struct values { t8 v[WIDE ? 1 : DT]; };
    __device__ __forceinline__ void values_of(values &x, uint32_t tl) const {
        if constexpr (!WIDE) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                s16x4 h[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t at = ((tl + voff) ^ (uint32_t) dt * 16u * DA) + 16u * i * L::ROWB;
                    h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *) (S + at));
                }
                x.v[dt] = __builtin_bit_cast(t8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
            }
        }
    }

    // O^T += V^T P^T for the tile at `tl`, from key `key` on.
    // CAREFUL: an infinite or NaN value must not reach rows that do not see its key
    // (0 times it is NaN): such values are left out of the products and added to
    // the rows that see them.
    template <bool CAREFUL>
    __device__ __forceinline__ void products(const values &x, const probs &p, uint32_t key, uint32_t tl) {
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    float vf = *reinterpret_cast<const float *>(S + ((tl + voff) ^ (uint32_t) dt * 16u * DA) + i * L::ROWB);
                    if (CAREFUL) vf = odd(vf) ? 0.0f : vf;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) o[dt][nt] = mfma(vf, p.w[nt][i], o[dt][nt]);
                }
            }
        } else {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                t8 vf = x.v[dt];
                if (CAREFUL) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) vf[e] = odd((float) vf[e]) ? (T) 0.0f : vf[e];
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    o[dt][nt] = mfma(vf, p.p[nt], o[dt][nt]);
                    if constexpr (MOREW > 0) o[dt][nt] = mfma(vf, p.rest[nt], o[dt][nt]);
                    if constexpr (MOREW > 1) o[dt][nt] = mfma(vf, p.last[nt], o[dt][nt]);
                }
            }
        }
        if (CAREFUL) {
            for (uint32_t r = 0; r < (uint32_t) KT; ++r) {
                const uint8_t *row = S + tl + L::VALUES + r * L::ROWB;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t by = (16u * dt + 4u * g + i) * (uint32_t) sizeof(T);
                        const float v = (float) *reinterpret_cast<const T *>(row + ((by >> 4) ^ L::vsw(r)) * 16u + (by & 15u));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            if (odd(v) && (int) (key + r) < lim[nt]) o[dt][nt][i] += v;
                        }
                    }
                }
            }
        }
    }

    __device__ __forceinline__ void clear(scores &s) const {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[ks][nt] = (f32x4) { 0, 0, 0, 0 };
        }
    }

    // the first of the wave's tiles; key0 is a tile's first key
    __device__ __forceinline__ uint32_t first_tile() const { return it.key0 / KT + (KEYS ? wave : 0u); }
    static constexpr uint32_t STEP = KEYS ? WAVES : 1;
    load x;                         // KEYS: the tile that is on its way

    __device__ __forceinline__ uint32_t stage(uint32_t b) const { return (KEYS ? wave : b) * L::BYTES; }
    // the first tiles set off
    __device__ __forceinline__ void start() {
        if (it.key0 >= it.key1) return;
        const uint32_t t = first_tile();
        if constexpr (HELD8) {
            set_off(t);
            if constexpr (!KEYS && SETS == 2) issue8<SETS - 1>(t + 1);
        } else if constexpr (KEYS) {
            fetch(x, spans(t), t);
        } else {
            issue(t, stage(0));
            issue(t + 1, stage(1));
        }
    }
    // 8 bits: tile t's codes, into registers
    __device__ __forceinline__ void set_off(uint32_t t) {
        if constexpr (KEYS) {
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) fetch8(c8[gr], rows_at(t * KT + (uint32_t) gr * GROUP), t * KT + (uint32_t) gr * GROUP);
        } else {
            issue8<0>(t);
        }
    }

    // KEYS: tile t, in registers, which then take the next (two tiles on their way at a
    // time were no faster: 58.8 us and 57.4 for 8 sequences of 16384 positions, bf16)
    template <bool CAREFUL>
    __device__ __forceinline__ void turn(uint32_t t) {
        const uint32_t then = t + STEP;
        scores s;
        clear(s);
        if constexpr (HELD8) {
            span m[GROUPS];
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) m[gr] = rows_at(then * KT + (uint32_t) gr * GROUP);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int j = 0; j < KL; ++j) {
                    const two k = widen(c8[ks].k[j], c8[ks].ks);
                    score<CAREFUL>(s[ks], k.p[0], 2 * j);
                    score<CAREFUL>(s[ks], k.p[1], 2 * j + 1);
                }
            }
#pragma unroll
            for (int gr = 0; gr < GROUPS; ++gr) land(c8[gr], stage(0) + gr * GROUP * L::ROWB);
            __builtin_amdgcn_sched_barrier(0);
            if (then * KT < it.key1) {
#pragma unroll
                for (int gr = 0; gr < GROUPS; ++gr) fetch8(c8[gr], m[gr], then * KT + (uint32_t) gr * GROUP);
            }
        } else {
        const span_of_tile m = spans(then);                      // (past the end: the last page again)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
            for (int q = 0; q < QC; ++q) score<CAREFUL>(s[ks], x.k[ks][q], q);
        }
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) {
#pragma unroll
            for (int j = 0; j < COPIES; ++j) *reinterpret_cast<u32x4 *>(S + stage(0) + vput[j] + gr * GROUP * L::ROWB) = x.v[gr][j];
        }
        __builtin_amdgcn_sched_barrier(0);
        if (then * KT < it.key1) fetch(x, m, then);
        }
        mask(s, t * KT);
        probs p;
        float f[NT];
        if (adjust(s, f)) rescale(f);
        soften(s, p);
        __builtin_amdgcn_sched_barrier(0);
        values v;
        values_of(v, stage(0));
        products<CAREFUL>(v, p, t * KT, stage(0));
    }

    template <bool CAREFUL>
    __device__ __forceinline__ void scores_of(scores &s, uint32_t at) const {
        clear(s);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
            for (int q = 0; q < QC; ++q) score<CAREFUL>(s[ks], *reinterpret_cast<const u32x4 *>(S + at + koff[q] + 16u * ks * L::ROWB), q);
        }
    }
    // not KEYS: all but the last N of the wave's loads have arrived, and the other
    // waves' have too; the stages read before are free
    template <int N> __device__ __forceinline__ void meet() const {
        wait_vmem<N>();
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }

    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = LOWEST;
            l[nt] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt][nt] = (f32x4) { 0, 0, 0, 0 };
        }
    }

    // The order of a loop iteration's instructions: the keys' reads, then each matrix
    // instruction with its share of the vector ones and of the values' reads. (2 to 8
    // vector instructions each: within 2 % of each other. Over 8 bits as if queries were one
    // piece: 4 times 512 f32 rows behind 4000 150.7 us, 156 by their true number.)
    __device__ __forceinline__ static void interleave() {
        constexpr int VECTOR = 4;
        constexpr int PER = (WIDE ? 4 : 1) * NT * (SPLIT ? 2 : 1);
        constexpr int MS = KS * QC * PER, MP = DT * PER, DV = WIDE ? 4 * DT : 0;
        __builtin_amdgcn_sched_group_barrier(0x100, KS * QC, 0);
#pragma unroll
        for (int i = 0; i < MS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x2, VECTOR, 0);
            if (i < DV) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
#pragma unroll
        for (int i = 0; i < MP; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x2, VECTOR, 0);
        }
    }

    // The keys of the range, once (start() went before). Not KEYS: three tiles are worked
    // on at a time, the scores of one, p of the one before it and the products of the one
    // before that, which do not wait for each other: the matrix unit and the vector unit
    // both have work. A tile's copy is asked for two tiles ahead.
    __device__ __forceinline__ void pass() {
        begin();
        if (it.key0 >= it.key1) return;
        const uint32_t t1 = (it.key1 + KT - 1u) / KT;
        uint32_t t = first_tile();
        if constexpr (KEYS) {
            for (; t < t1; t += STEP) turn<false>(t);
        } else if constexpr (HELD8) {
            pass8(t, t1);
        } else {
            scores s, next;
            probs p;
            float f[NT];
            meet<VM>();
            issue(t + 2, stage(2));
            scores_of<false>(s, stage(0));
            meet<VM>();
            scores_of<false>(next, stage(1));
            mask(s, t * KT);
            bool moved = adjust(s, f);
            soften(s, p);
            uint32_t n = 1;                                      // tile t + n's scores are `next`
            for (; t + n < t1; ++n) {
                if (moved) rescale(f);
                meet<0>();
                // (the transposing reads before the copy: the compiler waits for copies to LDS before one)
                values v;
                values_of(v, stage((n - 1) & 3u));
                __builtin_amdgcn_sched_barrier(0);
                issue(t + n + 2, stage((n + 2) & 3u));
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s[ks][nt] = next[ks][nt];
                }
                mask(s, (t + n) * KT);
                moved = adjust(s, f);                            // (the tile before it is still on its way into o)
                __builtin_amdgcn_sched_barrier(0);
                probs q;
                scores_of<false>(next, stage((n + 1) & 3u));
                products<false>(v, p, (t + n - 1) * KT, stage((n - 1) & 3u));
                soften(s, q);
                p = q;
                interleave();
            }
            if (moved) rescale(f);
            wait_vmem<0>();                                      // nothing comes into LDS any more
            values v;
            values_of(v, stage((n - 1) & 3u));
            products<false>(v, p, (t + n - 1) * KT, stage((n - 1) & 3u));
        }
    }

    // 8 bits: the same steps, but a tile comes into registers and is put into LDS an
    // iteration later, as T.
    __device__ __forceinline__ void meet8() const {
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
    // Tile t + n: the one two further comes out of registers into LDS, and the next into them.
    template <int B>
    __device__ __forceinline__ void step8(scores &s, scores &next, probs &p, float (&f)[NT], bool &moved, uint32_t t, uint32_t n) {
        if (moved) rescale(f);
        meet8();
        values v;
        values_of(v, stage((n - 1) & 3u));
        land(c8[B], stage((n + 2) & 3u));
        issue8<B>(t + n + 2 + SETS);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[ks][nt] = next[ks][nt];
        }
        mask(s, (t + n) * KT);
        moved = adjust(s, f);
        __builtin_amdgcn_sched_barrier(0);
        probs q;
        scores_of<false>(next, stage((n + 1) & 3u));
        products<false>(v, p, (t + n - 1) * KT, stage((n - 1) & 3u));
        soften(s, q);
        p = q;
        interleave();
    }
    __device__ __forceinline__ void pass8(const uint32_t t, const uint32_t t1) {
        scores s, next;
        probs p;
        float f[NT];
        constexpr int ODD = SETS - 1;                            // the registers of odd tiles
        land(c8[0], stage(0));                                   // (a tile past the end is zeros)
        issue8<0>(t + SETS);
        land(c8[ODD], stage(1));
        issue8<ODD>(t + 1 + SETS);
        land(c8[0], stage(2));
        issue8<0>(t + 2 + SETS);
        meet8();
        scores_of<false>(s, stage(0));
        scores_of<false>(next, stage(1));
        mask(s, t * KT);
        bool moved = adjust(s, f);
        soften(s, p);
        uint32_t n = 1;                                          // tile t + n's scores are `next`
        if constexpr (SETS == 2) {
            for (; t + n + 1 < t1; n += 2) {
                step8<ODD>(s, next, p, f, moved, t, n);
                step8<0>(s, next, p, f, moved, t, n + 1);
            }
        }
        for (; t + n < t1; ++n) step8<ODD>(s, next, p, f, moved, t, n);
        if (moved) rescale(f);
        values v;
        values_of(v, stage((n - 1) & 3u));
        products<false>(v, p, (t + n - 1) * KT, stage((n - 1) & 3u));
    }

    // The same with care, a tile after the other.
    __device__ __forceinline__ void careful_pass() {
        begin();
        if (it.key0 >= it.key1) return;
        const uint32_t t1 = (it.key1 + KT - 1u) / KT;
        for (uint32_t t = first_tile(); t < t1; t += STEP) {
            if constexpr (KEYS) {
                if constexpr (HELD8) set_off(t);
                else fetch(x, spans(t), t);
                turn<true>(t);
            } else {
                if constexpr (HELD8) {
                    set_off(t);
                    land(c8[0], stage(0));
                } else {
                    issue(t, stage(0));
                }
                meet<0>();
                scores s;
                probs p;
                values v;
                float f[NT];
                scores_of<true>(s, stage(0));
                mask(s, t * KT);
                if (adjust(s, f)) rescale(f);
                soften(s, p);
                values_of(v, stage(0));
                products<true>(v, p, t * KT, stage(0));
                meet<0>();
            }
        }
    }

    __device__ __forceinline__ bool has_odd() const {
        bool bad = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) bad |= odd(o[dt][nt][i]);
            }
        }
        return bad;
    }

    // where a row's results go, once for all its dimensions
    __device__ __forceinline__ uint8_t *out_row(uint32_t row) const {
        const place at = place_of(row);
        return (uint8_t *) a.out + token(at.t) * a.out_tok + at.h * a.out_head;
    }
    // four of them, as they are stored: 16 bits, a pair a register
    __device__ __forceinline__ static u32x2 packed(f32x4 x) {
        typename vec4<A>::type y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = (A) x[i];
        return __builtin_bit_cast(u32x2, y);
    }
    // four of them, from dimension d on
    __device__ __forceinline__ void put(uint8_t *dst, uint32_t d, f32x4 x) const {
        if (d >= a.hd) return;
        if constexpr (sizeof(A) == 4) *G_CAST(f32x4, dst + d * sizeof(A)) = x;
        else *G_CAST(u32x2, dst + d * sizeof(A)) = packed(x);
    }
    // Two dimension tiles of 16 bits: the lanes of a row swap, so that each has eight
    // values that are adjacent and a row's 64 bytes are written by one instruction.
    __device__ __forceinline__ void put_two(uint8_t *dst, int dt, f32x4 x0, f32x4 x1) const {
        const u32x2 p = packed(x0), q = packed(x1);
        const u32x2 lo = __builtin_amdgcn_permlane16_swap(p[0], q[0], false, false);
        const u32x2 hi = __builtin_amdgcn_permlane16_swap(p[1], q[1], false, false);
        const uint32_t d = 16u * ((uint32_t) dt + (g & 1u)) + 8u * (g >> 1);
        if (d < a.hd) *G_CAST(u32x4, dst + d * sizeof(A)) = (u32x4) { lo[0], hi[0], lo[1], hi[1] };
    }
    // a row of N times four results, STEP dimensions apart from d on
    template <int N, int STEP>
    __device__ __forceinline__ void finish(uint32_t row, uint32_t d, const f32x4 (&x)[N], float top, float sum, bool sees) const {
        if (it.part == ATT_DIRECT) {
            uint8_t *dst = out_row(row);
            const float by = sees ? 1.0f / sum : 0.0f;
            f32x4 y[N];
#pragma unroll
            for (int n = 0; n < N; ++n) y[n] = sees ? x[n] * by : (f32x4) { 0, 0, 0, 0 };
            if constexpr (sizeof(A) == 2 && N > 1) {             // (the four lanes of a row are here together)
#pragma unroll
                for (int n = 0; n < N; n += 2) put_two(dst, n, y[n], y[n + 1]);
            } else {
#pragma unroll
                for (int n = 0; n < N; ++n) put(dst, d + n * STEP, y[n]);
            }
        } else {
            const uint64_t at = it.part + row;
#pragma unroll
            for (int n = 0; n < N; ++n) *G_CAST(f32x4, a.part_o + at * D + d + n * STEP) = x[n];
            if (d == 0) {
                G_CAST(float, a.part_ml)[2 * at] = top;
                G_CAST(float, a.part_ml)[2 * at + 1] = sum;
            }
        }
    }

    __device__ __forceinline__ void run() {
        places();
        start();                                                 // the first tile is on its way while q is read
        load_q();
        pass();
        // 0 x inf in a key that a row does not see: only then is anything not finite
        // that need not be, and only then is the pass made again
        if (KEYS) {
            if (__any(has_odd())) careful_pass();
        } else {
            uint32_t *votes = reinterpret_cast<uint32_t *>(S + L::LDS);
            const bool bad = __any(has_odd());
            if (lane == 0) votes[wave] = bad;
            __syncthreads();
            if ((votes[0] | votes[1] | votes[2] | votes[3]) != 0) careful_pass();
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) l[nt] = row_sum(l[nt]);
        if constexpr (!KEYS) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint32_t row = wave * (16u * NT) + 16u * nt + li;
                if (row < it.n_rows) {
                    f32x4 x[DT];
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) x[dt] = o[dt][nt];
                    finish<DT, 16>(row, 4u * g, x, m[nt], l[nt], lim[nt] > 0);
                }
            }
        } else {
            // the waves' results side by side in LDS: [wave][row][D], then (m, l)
            __syncthreads();
            float *so = reinterpret_cast<float *>(S);
            float *sm = so + WAVES * 16 * NT * D;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint32_t row = wave * (16u * NT) + 16u * nt + li;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4 *>(so + row * D + 16 * dt + 4 * g) = o[dt][nt];
                if (g == 0) {
                    sm[2 * row] = m[nt];
                    sm[2 * row + 1] = l[nt];
                }
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < it.n_rows * (D / 4); i += ATT_THREADS) {
                const uint32_t row = i / (D / 4), d = 4u * (i % (D / 4));
                float top = LOWEST, sum = 0.0f, ml[WAVES][2];
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    ml[w][0] = sm[2 * (w * 16 * NT + row)];
                    ml[w][1] = sm[2 * (w * 16 * NT + row) + 1];
                    top = fmaxf(top, ml[w][0]);
                }
                f32x4 x[1] = { { 0, 0, 0, 0 } };
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    const float f = __builtin_amdgcn_exp2f(ml[w][0] - top);
                    sum += f * ml[w][1];
                    x[0] += f * *reinterpret_cast<const f32x4 *>(so + (w * 16 * NT + row) * D + d);
                }
                finish<1, 0>(row, d, x, top, sum, limit(place_of(row).t) > 0);
            }
        }
    }
};

template <typename A, typename T, int D, int NT, bool KEYS, bool PAGED, typename C = T>
__device__ __forceinline__ void attend_item(const att_args &a, const att_item &it, uint8_t *S) {
    const uint32_t lane = threadIdx.x & 63u;
    attention<A, T, D, NT, KEYS, PAGED, C> x = { a, it, S, lane, uniform(threadIdx.x >> 6), lane >> 4, lane & 15u };
    x.run();
}

// One LDS variable a kernel: beside a second, the compiler waits for copies to the one
// before it reads it anywhere.
constexpr int VOTES = WAVES * 4;
constexpr int max_of(int a, int b) { return a > b ? a : b; }
template <typename T, int D> constexpr int LDS_BYTES =
    max_of(max_of(tile<T, D, false>::LDS + VOTES, tile<T, D, true>::LDS), WAVES * ATT_FEW_ROWS * (D + 2) * 4);

__device__ __forceinline__ att_item item_of(const att_args &a) {
    att_item it;
    uint32_t w[sizeof(att_item) / 4];
#pragma unroll
    for (uint32_t i = 0; i < sizeof(att_item) / 4; ++i) w[i] = C_CAST(uint32_t, a.items + blockIdx.x)[i];
    __builtin_memcpy(&it, w, sizeof it);
    return it;
}

// Whole prompts. 4 head_dim operations for a row and a key that it sees: the matrix unit
// bounds f32, the vector unit beside it 16 bits (3.8 instructions to a matrix one, of
// which one in seven is an exponential). Two workgroups a CU, 64 KB of LDS and at most 256
// registers each, so that one's barrier falls into the other's products; 128 rows a
// workgroup read a tile of keys from LDS once for two products. With 20 heads over 5 of
// 128: 16384 rows f16 1.40 to 1.50 ms by machine, 0.92 to 0.98 PFLOP/s (a large product
// reaches 1.20; the clock goes down to about 1.9 GHz under both); 24 prompts of up to 2048
// rows bf16 149 to 155 us, 0.66 to 0.69, where reading q and writing the results (37 us of
// copying) is little hidden; 4 prompts f32 497 us, 110 TFLOP/s of 153, the matrix unit busy
// 81 % of the time. 32 rows a wave and not 64, one wave a SIMD: 1.52 against 1.85 ms. A
// head_dim is padded to 64 or 128: 4096 rows bf16 take 85 us at 64, 117 at 80, 118 at 96
// (no tile's rows are whole there, so each copy asks) and 112 at 128.
template <typename T, int D>
__device__ __forceinline__ void prompt_body(const att_args &a) {
    __shared__ __attribute__((aligned(1024))) uint8_t S[LDS_BYTES<T, D>];
    const att_item it = item_of(a);
    if (it.mode == ATT_FEW) attend_item<T, T, D, 1, true, false>(a, it, S);
    else if (it.mode == ATT_HALF) attend_item<T, T, D, 1, false, false>(a, it, S);
    else attend_item<T, T, D, 2, false, false>(a, it, S);
}

// A step over the cache. Few rows (one sequence's own keys) are bound by memory: each
// key is read once, straight into registers, by one wave, and a split's four waves are
// joined in LDS. 8 sequences of up to 65536 positions, bf16, 20 heads over 5 of 128: 374
// MB in 63.0 us with the join, 5.9 TB/s. Many rows (keys that sequences share, prompts
// behind a prefix) go as prompts do: 64 sequences behind 4096 shared positions and up to
// 1024 of their own, f32 rows over f16, 30.1 us. All kinds in one launch, so
// that few and many rows run side by side: at these sizes a workgroup's start, the
// uneven shares and the join's launch bound it.
template <typename A, typename T, int D>
__device__ __forceinline__ void paged_body(const att_args &a) {
    __shared__ __attribute__((aligned(1024))) uint8_t S[LDS_BYTES<T, D>];
    const att_item it = item_of(a);
    if (it.mode == ATT_FEW) attend_item<A, T, D, 1, true, true>(a, it, S);
    else if (it.mode == ATT_HALF) attend_item<A, T, D, 1, false, true>(a, it, S);
    else attend_item<A, T, D, 2, false, true>(a, it, S);
}

// The same over 8 bits: codes come into registers, half the bytes of bf16, and are turned into bf16
// there: for few rows right before the products, else once for a workgroup on the way to LDS. A
// scale is a power of two, so nothing is rounded and no score or weight is multiplied by it. What
// that costs the vector unit, 2.75 instructions a value of int8 and half of one of e4m3, memory hides
// for few rows: 8 sequences of up to 65536 positions, e4m3 under bf16, 317 MB in 58.1 us with the join,
// 5.4 TB/s (without the loads of scales it would be 56.4). Many rows are bound as over bf16: 64
// sequences behind 4096 shared positions, int8, 24.8 us; one of 1101 positions, f32 rows, 9.3 us, two
// launches. Two tiles of few rows on their way at a time: 57.9 us for 58.6, but 26.8 for 26.0 behind a shared
// prefix. (Queries of f32 take three times the registers: no 32 rows a wave.)
template <typename A, typename C, int D>
__device__ __forceinline__ void held8_body(const att_args &a) {
    __shared__ __attribute__((aligned(1024))) uint8_t S[LDS_BYTES<__bf16, D>];
    const att_item it = item_of(a);
    if (it.mode == ATT_FEW) attend_item<A, __bf16, D, 1, true, true, C>(a, it, S);
    else if (sizeof(A) == 4 || it.mode == ATT_HALF) attend_item<A, __bf16, D, 1, false, true, C>(a, it, S);
    else if constexpr (sizeof(A) == 2) attend_item<A, __bf16, D, 2, false, true, C>(a, it, S);
}

}  // namespace

#define PROMPT(name, T, D) extern "C" __global__ void __launch_bounds__(ATT_THREADS, 2) name(const att_args a) { prompt_body<T, D>(a); }
#define PAGED(name, A, T, D) extern "C" __global__ void __launch_bounds__(ATT_THREADS, 2) name(const att_args a) { paged_body<A, T, D>(a); }

#define HELD8(name, A, C)                                                                                                                                   \
    extern "C" __global__ void __launch_bounds__(ATT_THREADS, 2) sllm_k_attend_##name##_64(const att_args a) { held8_body<A, C, 64>(a); }        \
    extern "C" __global__ void __launch_bounds__(ATT_THREADS, 2) sllm_k_attend_##name##_128(const att_args a) { held8_body<A, C, 128>(a); }

HELD8(f32i8, float, int8_codes)
HELD8(f16i8, _Float16, int8_codes)
HELD8(bf16i8, __bf16, int8_codes)
HELD8(f32e4m3, float, e4m3_codes)
HELD8(f16e4m3, _Float16, e4m3_codes)
HELD8(bf16e4m3, __bf16, e4m3_codes)
PAGED(sllm_k_attend_f32_64, float, float, 64)
PAGED(sllm_k_attend_f32_128, float, float, 128)
PAGED(sllm_k_attend_f32f16_64, float, _Float16, 64)
PAGED(sllm_k_attend_f32f16_128, float, _Float16, 128)
PAGED(sllm_k_attend_f16_64, _Float16, _Float16, 64)
PAGED(sllm_k_attend_f16_128, _Float16, _Float16, 128)
PAGED(sllm_k_attend_bf16_64, __bf16, __bf16, 64)
PAGED(sllm_k_attend_bf16_128, __bf16, __bf16, 128)
PROMPT(sllm_k_prompt_f32_64, float, 64)
PROMPT(sllm_k_prompt_f32_128, float, 128)
PROMPT(sllm_k_prompt_f16_64, _Float16, 64)
PROMPT(sllm_k_prompt_f16_128, _Float16, 128)
PROMPT(sllm_k_prompt_bf16_64, __bf16, 64)
PROMPT(sllm_k_prompt_bf16_128, __bf16, 128)

namespace {

// The partial results of one row: out = sum_i f_i o_i / sum_i f_i l_i with f_i =
// 2^(m_i - M), M the largest m_i, added up in an order that the split alone gives,
// so that the same call gives the same bits. WHOLE: a workgroup a row, its waves
// taking every fourth split of a segment; else a wave a row. What costs is the chain
// of loads (token, segment, parts): a part's o, m and l are asked for together, and
// several splits at once. 5120 rows of up to 4 parts, a wave each, 4.9 us; 1280 rows of
// about 10, a workgroup each, 5.0 us; 20 rows of 18 parts 3.4 us.
template <typename A, int D, bool WHOLE>
__device__ __forceinline__ void join_body(const att_join_args &a) {
    constexpr int V = D / 64, UN = 4;
    typedef float vec __attribute__((ext_vector_type(V)));
    const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6);
    const uint32_t tok = blockIdx.x, h = WHOLE ? blockIdx.y : blockIdx.y * WAVES + wave;
    if (h >= a.n_head) return;
    const uint32_t kvh = h / a.group, hh = h % a.group;
    const uint32_t seg0 = C_CAST(uint32_t, &a.toks[tok].seg0)[0], n_seg = C_CAST(uint32_t, &a.toks[tok].n_seg)[0];
    const uint32_t at = C_CAST(uint32_t, &a.toks[tok].t)[0] * a.group + hh;
    if (n_seg == 0) return;                                      // written already
    constexpr uint32_t STEP = WHOLE ? WAVES : 1;
    float top = LOWEST, sum = 0.0f, x[V] = {};
    for (uint32_t i = 0; i < n_seg; ++i) {
        const uint32_t part0 = C_CAST(uint32_t, &a.segs[seg0 + i].part0)[0], n_rows = C_CAST(uint32_t, &a.segs[seg0 + i].n_rows)[0];
        const uint32_t n_split = C_CAST(uint32_t, &a.segs[seg0 + i].n_split)[0], off = C_CAST(uint32_t, &a.segs[seg0 + i].row_off)[0];
        const uint64_t row = part0 + (uint64_t) kvh * n_split * n_rows + off + at;
        for (uint32_t k = WHOLE ? wave : 0u; k < n_split; k += STEP * UN) {
            float m[UN], l[UN];
            vec o[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {                       // (past the end: the last split again, with no weight)
                const uint64_t r = row + (uint64_t) min(k + (uint32_t) u * STEP, n_split - 1u) * n_rows;
                m[u] = G_CAST(const float, a.part_ml)[2 * r];
                l[u] = G_CAST(const float, a.part_ml)[2 * r + 1];
                o[u] = *G_CAST(const vec, a.part_o + r * D + V * lane);
            }
            float up = top;
#pragma unroll
            for (int u = 0; u < UN; ++u) up = fmaxf(up, m[u]);
            const float f = __builtin_amdgcn_exp2f(top - up);
            top = up;
            sum *= f;
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] *= f;
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                if (k + (uint32_t) u * STEP < n_split) {
                    const float e = __builtin_amdgcn_exp2f(m[u] - up);
                    sum = fmaf(l[u], e, sum);
#pragma unroll
                    for (int v = 0; v < V; ++v) x[v] = fmaf(o[u][v], e, x[v]);
                }
            }
        }
    }
    A *out = (A *) ((uint8_t *) a.out + tok * a.out_tok) + (uint64_t) h * a.hd;
    if constexpr (!WHOLE) {
        if (V * lane < a.hd) {
#pragma unroll
            for (int v = 0; v < V; ++v) G_CAST(A, out)[V * lane + v] = (A) (x[v] / sum);
        }
    } else {
        __shared__ float so[WAVES][D], sm[WAVES][2];
#pragma unroll
        for (int v = 0; v < V; ++v) so[wave][V * lane + v] = x[v];
        if (lane == 0) {
            sm[wave][0] = top;
            sm[wave][1] = sum;
        }
        __syncthreads();
        if (threadIdx.x >= a.hd) return;
        float all = fmaxf(fmaxf(sm[0][0], sm[1][0]), fmaxf(sm[2][0], sm[3][0])), l = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float e = __builtin_amdgcn_exp2f(sm[w][0] - all);
            l = fmaf(sm[w][1], e, l);
            o = fmaf(so[w][threadIdx.x], e, o);
        }
        G_CAST(A, out)[threadIdx.x] = (A) (o / l);
    }
}

// A step's rows into their pages: a thread for each eight values of a row,
// blockIdx.y the KV head's keys or values, so that a wave writes whole lines of a page.
// Bound by memory: 18355 rows f32 to f16, 5 KV heads of 128, 29.7 us, 4.7 TB/s read and
// written; a step of 64 rows is its launch, 2.5 us.
template <typename A, typename T>
__device__ __forceinline__ void store_body(const att_store_args &a) {
    const uint32_t per_row = a.hd / 8, id = blockIdx.x * ATT_THREADS + threadIdx.x;
    const uint32_t tok = id / per_row, ch = id % per_row, h = blockIdx.y >> 1, kv = blockIdx.y & 1u;
    if (tok >= a.n_tok) return;
    const uint32_t pos = a.toks[tok].pos, page = a.tables[a.toks[tok].table + (pos >> a.page_shift)];
    const uint8_t *src = kv ? (const uint8_t *) a.v + tok * a.v_tok : (const uint8_t *) a.k + tok * a.k_tok;
    src += (h * a.hd + 8u * ch) * sizeof(A);
    uint8_t *dst = (kv ? a.cv : a.ck) + page * a.page_bytes +
                   (((uint64_t) (h << a.page_shift) + (pos & ((1u << a.page_shift) - 1u))) * a.hd + 8u * ch) * sizeof(T);
    if constexpr (sizeof(A) == sizeof(T)) {
#pragma unroll
        for (int i = 0; i < (int) sizeof(T) / 2; ++i) G_CAST(u32x4, dst)[i] = G_CAST(const u32x4, src)[i];
    } else {
        typename vec8<T>::type y;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x4 x = G_CAST(const f32x4, src)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[4 * i + e] = (T) x[e];    // to nearest, ties to even
        }
        *G_CAST(u32x4, dst) = __builtin_bit_cast(u32x4, y);
    }
}

}  // namespace

#define JOIN(name, A, D)                                                                                                                  \
    extern "C" __global__ void __launch_bounds__(ATT_THREADS) name(const att_join_args a) { join_body<A, D, false>(a); }                  \
    extern "C" __global__ void __launch_bounds__(ATT_THREADS) name##_whole(const att_join_args a) { join_body<A, D, true>(a); }
#define STORE(name, A, T) extern "C" __global__ void __launch_bounds__(ATT_THREADS) name(const att_store_args a) { store_body<A, T>(a); }

JOIN(sllm_k_attn_join_f32_64, float, 64)
JOIN(sllm_k_attn_join_f32_128, float, 128)
JOIN(sllm_k_attn_join_f16_64, _Float16, 64)
JOIN(sllm_k_attn_join_f16_128, _Float16, 128)
JOIN(sllm_k_attn_join_bf16_64, __bf16, 64)
JOIN(sllm_k_attn_join_bf16_128, __bf16, 128)
STORE(sllm_k_attn_store_f32, float, float)
STORE(sllm_k_attn_store_f32f16, float, _Float16)
STORE(sllm_k_attn_store_16, _Float16, _Float16)

namespace {

// Pages to pages: blockIdx.y a pair of them, ATT_COPY_CHUNKS 16-byte pieces of
// what it holds a workgroup, all four of a thread's in flight together. Bound by
// memory: 396 pages of 655 KB moved or copied in two launches 92 us, 5.5 TB/s; 16 copies
// of 41 positions of 30 layers, a source that the caches hold, 15.2 us, 3.5 TB/s.
// SCALES: of each block also the scale bytes of those rows, the last of them one by one.
template <bool SCALES> __device__ __forceinline__ void copy_body(const att_copy_args &a) {
    att_pair p;
    if (a.list) p = { C_CAST(uint32_t, a.list + blockIdx.y)[0], C_CAST(uint32_t, a.list + blockIdx.y)[1], C_CAST(uint32_t, a.list + blockIdx.y)[2] };
    else p = a.pair[blockIdx.y];
    const uint32_t codes = p.rows * a.row_bytes / 16u, per = codes + (SCALES ? (p.rows + 15u) / 16u : 0u), n = per * a.n_blocks;
    const uint8_t *src = a.mem + p.src * a.page_bytes;
    uint8_t *dst = a.mem + p.dst * a.page_bytes;
    constexpr int UN = ATT_COPY_CHUNKS / ATT_THREADS;
    u32x4 v[UN];
    uint64_t at[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
        const uint32_t x = blockIdx.x * ATT_COPY_CHUNKS + (uint32_t) i * ATT_THREADS + threadIdx.x;
        const uint32_t y = x % per;
        at[i] = (uint64_t) (x / per) * a.block_bytes + (!SCALES || y < codes ? y * 16u : a.scales + (y - codes) * 16u);
        if (x < n) v[i] = *G_CAST(const u32x4, src + at[i]);
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
        const uint32_t x = blockIdx.x * ATT_COPY_CHUNKS + (uint32_t) i * ATT_THREADS + threadIdx.x;
        if (x >= n) return;
        if constexpr (SCALES) {
            const uint32_t y = x % per, left = y < codes ? 16u : p.rows - (y - codes) * 16u;
            if (left < 16u) {
#pragma unroll
                for (uint32_t j = 0; j < 15u; ++j) if (j < left) G_CAST(uint8_t, dst + at[i])[j] = (uint8_t) (v[i][j >> 2] >> (8u * (j & 3u)));
                continue;
            }
        }
        *G_CAST(u32x4, dst + at[i]) = v[i];
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(ATT_THREADS) sllm_k_attn_copy(const att_copy_args a) { copy_body<false>(a); }
extern "C" __global__ void __launch_bounds__(ATT_THREADS) sllm_k_attn_copy8(const att_copy_args a) { copy_body<true>(a); }

// ---------------------------------------------------------------------------
// rows on their way: rotary positions, a cache of 8 bits
// ---------------------------------------------------------------------------

namespace {

// cos and sin of p / 2^32 turns: the quarter turn that p is nearest to, and the two series
// on what is left, |x| <= pi / 4 (the first terms left out are x^13 / 13! and x^12 / 12!,
// under 2^-32). p is exact to 2 of 2^-32 turns however far the position; what is left of it is
// rounded to f32 (up to 2^-28 of a turn) and again by its product.
__device__ __forceinline__ void cos_sin(uint32_t p, float &c, float &s) {
    const uint32_t quarter = (p + 0x20000000u) >> 30;
    const float x = (float) (int32_t) (p - (quarter << 30)) * 1.46291807926715968e-9f, x2 = x * x;      // 2 pi / 2^32
    float a = fmaf(x2, -2.50521083854417188e-8f, 2.75573192239858907e-6f);
    a = fmaf(x2, a, -1.98412698412698413e-4f);
    a = fmaf(x2, a, 8.33333333333333333e-3f);
    a = fmaf(x2, a, -1.66666666666666667e-1f);
    a = fmaf(x2 * x, a, x);
    float b = fmaf(x2, -2.75573192239858907e-7f, 2.48015873015873016e-5f);
    b = fmaf(x2, b, -1.38888888888888889e-3f);
    b = fmaf(x2, b, 4.16666666666666667e-2f);
    b = fmaf(x2, b, -0.5f);
    b = fmaf(x2, b, 1.0f);
    c = quarter & 1u ? a : b;
    s = quarter & 1u ? b : a;
    c = quarter == 1u || quarter == 2u ? -c : c;
    s = quarter >= 2u ? -s : s;
}

// eight values in two halves of four, at d0 and d1
template <typename A> struct eight {
    f32x4 x[2];
    __device__ __forceinline__ static f32x4 wide(u32x2 v) {
        const typename vec4<A>::type y = __builtin_bit_cast(typename vec4<A>::type, v);
        return (f32x4) { (float) y[0], (float) y[1], (float) y[2], (float) y[3] };
    }
    __device__ __forceinline__ void load(const uint8_t *row, uint32_t d0, uint32_t d1, bool whole) {
        if constexpr (sizeof(A) == 4) {
            x[0] = *G_CAST(const f32x4, row + d0 * 4u);
            x[1] = *G_CAST(const f32x4, row + d1 * 4u);
        } else if (whole) {
            const u32x4 v = *G_CAST(const u32x4, row + d0 * 2u);
            x[0] = wide((u32x2) { v[0], v[1] });
            x[1] = wide((u32x2) { v[2], v[3] });
        } else {
            x[0] = wide(*G_CAST(const u32x2, row + d0 * 2u));
            x[1] = wide(*G_CAST(const u32x2, row + d1 * 2u));
        }
    }
    __device__ __forceinline__ void store(uint8_t *row, uint32_t d0, uint32_t d1, bool whole) const {
        if constexpr (sizeof(A) == 4) {
            *G_CAST(f32x4, row + d0 * 4u) = x[0];
            *G_CAST(f32x4, row + d1 * 4u) = x[1];
        } else {
            u32x2 y[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                typename vec4<A>::type h;
#pragma unroll
                for (int e = 0; e < 4; ++e) h[e] = (A) x[i][e];
                y[i] = __builtin_bit_cast(u32x2, h);
            }
            if (whole) {
                *G_CAST(u32x4, row + d0 * 2u) = (u32x4) { y[0][0], y[0][1], y[1][0], y[1][1] };
            } else {
                *G_CAST(u32x2, row + d0 * 2u) = y[0];
                *G_CAST(u32x2, row + d1 * 2u) = y[1];
            }
        }
    }
};

template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, CTRL, 0xf, 0xf, true);
}

// A row's largest magnitude, as bits, over the 8 or 16 lanes that hold it (infinities and
// NaN are larger than all others).
__device__ __forceinline__ uint32_t top_of(const f32x4 (&x)[2], bool in, bool wide) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max(m, __float_as_uint(x[i][e]) & 0x7fffffffu);
    }
    m = in ? m : 0u;
    m = max(m, dpp<0xb1>(m));                                    // lane ^ 1
    m = max(m, dpp<0x4e>(m));                                    // lane ^ 2
    m = max(m, dpp<0x141>(m));                                   // 7 - lane, of eight
    return wide ? max(m, dpp<0x128>(m)) : m;                     // 8 further, of sixteen
}

// The scale byte of a row of that largest magnitude: the smallest 2^e, e >= -126 (e4m3:
// -117), with top <= 127 2^e (448 2^e), whose values are all normal f32 and bf16. Up to 127 2^120.
__device__ __forceinline__ uint32_t scale_of(uint32_t top, bool i8) {
    if (top > 0x7efe0000u) return ATT_NAN_ROW;
    const int e = (int) (top >> 23), m = (int) (top & 0x7fffffu);
    return (uint32_t) (i8 ? max(e - 6 + (m > 0x7e0000), 1) : max(e - 8 + (m > 0x600000), 10));
}
// four of a row's codes, each rounded once to the nearest, ties to even (a product with a
// power of two is exact, or so small that its code is 0)
__device__ __forceinline__ uint32_t codes_of(f32x4 x, uint32_t scale, bool i8) {
    if (scale == ATT_NAN_ROW) return i8 ? 0u : 0x7f7f7f7fu;
    const float by = __uint_as_float((254u - scale) << 23);
    if (i8) {
        uint32_t y = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) y |= ((uint32_t) (int) __builtin_rintf(x[e] * by) & 255u) << (8 * e);
        return y;
    }
    int y = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * by, x[1] * by, 0, false);
    return (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * by, x[3] * by, y, true);
}

// A lane's values of row h of a token's: queries, keys, values.
template <typename A>
__device__ __forceinline__ eight<A> row_of_token(const uint8_t *q, const uint8_t *k, const uint8_t *v, uint32_t h, uint32_t nq, uint32_t nk, uint32_t rows,
                                                 uint32_t hd, uint32_t unit, uint32_t d0, uint32_t d1, bool in, bool whole) {
    const bool is_q = h < nq, is_v = h >= nq + nk;
    const uint8_t *src = is_q ? q : is_v ? v : k;
    eight<A> x;
    x.x[0] = x.x[1] = (f32x4) { 0, 0, 0, 0 };
    if (h < rows && in) x.load(src + (uint64_t) (h - (is_q ? 0u : is_v ? nq + nk : nq)) * hd * sizeof(A), is_v ? 8u * unit : d0, is_v ? 8u * unit + 4u : d1, whole);
    return x;
}

// A wave takes the heads of one token, four rows of up to 128 values at a time (eight of up
// to 64), eight values a lane; cos and sin of a lane's four pairs are formed once for all of
// them. So a token's rows are read and written once, and nothing crosses lanes but a row's
// largest magnitude. Bound by memory: 18355 tokens of 20 + 5 heads of 128, bf16, turned, 235 MB in
// 48.5 us, 4.85 TB/s; their f32 keys and values to int8 24 us, 5.0 TB/s; 4099 tokens of 40 heads of
// 96, f16, 14.4 us. One token is its launch, 2.6 us (3.2 with the loads behind the angles).
template <typename A>
__device__ __forceinline__ void rows_body(const att_rows_args &a) {
    const uint32_t lane = threadIdx.x & 63u, w = blockIdx.x * (ATT_THREADS / 64) + uniform(threadIdx.x >> 6);
    const uint32_t tok = w / a.waves, part = w % a.waves;
    if (tok >= a.n_tok) return;
    const bool wide = a.hd > 64;
    const uint32_t per = wide ? 16u : 8u, at_once = 64u / per, unit = lane & (per - 1u);
    const bool in = unit < a.hd / 8u, turned = unit < a.half / 4u, whole = a.pairs != 0 || a.half == 0;
    // the dimensions of the lane's values, of rows that turn
    const uint32_t d0 = turned && !whole ? 4u * unit : 8u * unit, d1 = turned && !whole ? a.half + 4u * unit : 8u * unit + 4u;
    const int32_t pos = a.toks ? C_CAST(int32_t, &a.toks[tok].pos)[0] : a.pos ? C_CAST(int32_t, a.pos)[tok] : 0;
    uint64_t place = 0;                                          // the token's row of KV head 0 in the cache
    uint32_t slot = 0;
    if (a.ck) {
        slot = (uint32_t) pos & ((1u << a.page_shift) - 1u);
        place = C_CAST(uint32_t, a.tables)[C_CAST(uint32_t, &a.toks[tok].table)[0] + ((uint32_t) pos >> a.page_shift)] * a.page_bytes;
    }
    const bool held8 = a.held >= ATT_HELD_I8;
    // (copies: a choice between two of the arguments would put them all into scratch memory)
    const uint8_t *q = (const uint8_t *) a.q + tok * a.q_tok, *k = (const uint8_t *) a.k + tok * a.k_tok, *v = (const uint8_t *) a.v + tok * a.v_tok;
    uint8_t *qo = (uint8_t *) a.q_out + tok * a.qo_tok, *ko = (uint8_t *) a.k_out + tok * a.ko_tok, *ck = a.ck + place, *cv = a.cv + place;
    const uint32_t nq = a.q ? a.n_head : 0u, nk = a.k ? a.n_head_kv : 0u, nv = a.v ? a.n_head_kv : 0u, rows = nq + nk + nv;
    // (the next rows are on their way while some are worked on, the first while the angles are)
    eight<A> next = row_of_token<A>(q, k, v, part * at_once + lane / per, nq, nk, rows, a.hd, unit, d0, d1, in, whole);
    float c[4] = { 1.0f, 1.0f, 1.0f, 1.0f }, s[4] = {};
    if (turned && in) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t f = G_CAST(const uint64_t, a.freq)[4u * unit + j];
            cos_sin((uint32_t) ((f * (uint64_t) (int64_t) pos) >> 32), c[j], s[j]);
            c[j] *= a.magnitude;
            s[j] *= a.back ? -a.magnitude : a.magnitude;
        }
    }
    for (uint32_t r = part * at_once; r < rows; r += a.waves * at_once) {
        uint32_t h = r + lane / per;
        const bool here = h < rows && in;
        const bool is_q = h < nq, is_v = h >= nq + nk;
        h -= is_q ? 0u : is_v ? nq + nk : nq;
        // (values are not turned: a lane's are side by side)
        const uint32_t e0 = is_v ? 8u * unit : d0, e1 = is_v ? 8u * unit + 4u : d1;
        eight<A> x = next;
        next = row_of_token<A>(q, k, v, r + a.waves * at_once + lane / per, nq, nk, rows, a.hd, unit, d0, d1, in, whole);
        if (turned && !is_v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 lo = x.x[0], hi = x.x[1], near = j < 2 ? lo : hi;
                const float n0 = near[2 * (j & 1)], n1 = near[2 * (j & 1) + 1], f0 = lo[j], f1 = hi[j];
                const float u = whole ? n0 : f0, v = whole ? n1 : f1;
                const float p = fmaf(u, c[j], -(v * s[j])), q = fmaf(v, c[j], u * s[j]);
                if (whole) {
                    x.x[j >> 1][2 * (j & 1)] = p;
                    x.x[j >> 1][2 * (j & 1) + 1] = q;
                } else {
                    x.x[0][j] = p;
                    x.x[1][j] = q;
                }
            }
        }
        if (is_q || (!is_v && a.k_out)) {
            uint8_t *dst = is_q ? qo : ko;
            if (here) x.store(dst + (uint64_t) h * a.hd * sizeof(A), e0, e1, whole);
        }
        if (a.ck == nullptr) continue;
        uint8_t *block = is_v ? cv : ck;
        if (held8) {
            const bool i8 = a.held == ATT_HELD_I8;
            const uint32_t scale = scale_of(top_of(x.x, here, wide), i8);      // (every lane is here)
            if (!here || is_q) continue;
            block += (uint64_t) h * a.block_bytes;
            uint8_t *dst = block + slot * a.hd;
            const uint32_t y0 = codes_of(x.x[0], scale, i8), y1 = codes_of(x.x[1], scale, i8);
            if (whole) {
                *G_CAST(u32x2, dst + e0) = (u32x2) { y0, y1 };
            } else {
                *G_CAST(uint32_t, dst + e0) = y0;
                *G_CAST(uint32_t, dst + e1) = y1;
            }
            if (unit == 0) *G_CAST(uint8_t, block + (a.hd << a.page_shift) + slot) = (uint8_t) scale;
        } else if (here && !is_q) {
            const uint64_t at = ((uint64_t) (h << a.page_shift) + slot) * a.hd;
            if constexpr (sizeof(A) == 4) {
                if (a.held == ATT_HELD_F16) {
                    eight<_Float16> y;
                    y.x[0] = x.x[0];
                    y.x[1] = x.x[1];
                    y.store(block + at * 2u, e0, e1, whole);
                    continue;
                }
            }
            x.store(block + at * sizeof(A), e0, e1, whole);
        }
    }
}

}  // namespace

namespace {

// A batch's positions out of their pages. A workgroup's pieces of eight values are of one page;
// whose page it is, is searched for 64 sequences at a time. Bound by memory: 19000 positions of
// int8 to f32, 5 KV heads of 128, 25.5 us, 4.8 TB/s; 200 positions 3.9 us, which is the chain of loads from
// the sequence to the codes.
template <typename A>
__device__ __forceinline__ void read_body(const att_read_args &a) {
    const uint32_t lane = threadIdx.x & 63u, entry = blockIdx.x;
    const uint64_t page = (uint64_t) C_CAST(uint32_t, a.tables)[entry] * a.page_bytes;
    uint32_t lo = 0, n = a.n_seq;                                // the last of n sequences from lo on whose pages start at or before it
    while (n > 1) {
        const uint32_t step = (n + 63u) / 64u, at = lo + lane * step;
        const bool before = lane * step < n && G_CAST(const att_seq, a.seqs)[at].table <= entry;
        const uint32_t last = (uint32_t) __popcll(__ballot(before)) - 1u;
        lo += last * step;
        n = min(step, n - last * step);
    }
    lo = uniform(lo);
    const uint32_t first = C_CAST(uint32_t, &a.seqs[lo].table)[0], row0 = C_CAST(uint32_t, &a.seqs[lo].row0)[0];
    const uint32_t end = C_CAST(uint32_t, &a.seqs[lo + 1].row0)[0], start = row0 + ((entry - first) << a.page_shift);
    const uint32_t page_rows = 1u << a.page_shift, n_rows = min(end - start, page_rows);
    const uint32_t per = a.hd / 8u, per_block = n_rows * per, all = per_block * 2u * a.n_head_kv;
    const uint32_t base = blockIdx.y * (ATT_THREADS * ATT_READ_UNITS) + threadIdx.x;
#pragma unroll
    for (uint32_t i = 0; i < ATT_READ_UNITS; ++i) {
        const uint32_t x = base + i * ATT_THREADS;
        if (x >= all) return;
        const uint32_t b = x / per_block, y = x % per_block, row = y / per, d = 8u * (y % per);
        const bool v = b >= a.n_head_kv;
        const uint32_t h = v ? b - a.n_head_kv : b;
        const uint8_t *src = (v ? a.cv : a.ck) + page;
        uint8_t *dst = (uint8_t *) (v ? a.v : a.k) + (uint64_t) (start + row) * (v ? a.v_tok : a.k_tok) + (uint64_t) (h * a.hd + d) * sizeof(A);
        if (a.held >= ATT_HELD_I8) {
            src += (uint64_t) h * a.block_bytes;
            const u32x2 codes = *G_CAST(const u32x2, src + row * a.hd + d);
            const float by = scale_value(*G_CAST(const uint8_t, src + (a.hd << a.page_shift) + row));
            eight<A> z;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const u32x2 w = a.held == ATT_HELD_I8 ? values_of_codes<int8_codes>(codes[e], by) : values_of_codes<e4m3_codes>(codes[e], by);
                z.x[e] = (f32x4) { __uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u) };
            }
            z.store(dst, 0, 4, true);
        } else {
            const uint64_t at = ((uint64_t) (h << a.page_shift) + row) * a.hd + d;
            if constexpr (sizeof(A) == 4) {
                if (a.held == ATT_HELD_F16) {
                    eight<_Float16> z;
                    z.load(src + at * 2u, 0, 4, true);
                    eight<float> f;
                    f.x[0] = z.x[0];
                    f.x[1] = z.x[1];
                    f.store(dst, 0, 4, true);
                    continue;
                }
            }
            eight<A> z;
            z.load(src + at * sizeof(A), 0, 4, true);
            z.store(dst, 0, 4, true);
        }
    }
}

}  // namespace

#define ROWS(name, A) extern "C" __global__ void __launch_bounds__(ATT_THREADS) name(const att_rows_args a) { rows_body<A>(a); }
#define READ(name, A) extern "C" __global__ void __launch_bounds__(ATT_THREADS) name(const att_read_args a) { read_body<A>(a); }

ROWS(sllm_k_attn_rows_f32, float)
ROWS(sllm_k_attn_rows_f16, _Float16)
ROWS(sllm_k_attn_rows_bf16, __bf16)
READ(sllm_k_attn_read_f32, float)
READ(sllm_k_attn_read_f16, _Float16)
READ(sllm_k_attn_read_bf16, __bf16)

// ---------------------------------------------------------------------------
// beams
// ---------------------------------------------------------------------------

namespace {

// A logit and its token as a number that is larger where it comes first: by value, then the
// lower token. 0 is none.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
    uint32_t u = __float_as_uint(x);
    u = u == 0x80000000u ? 0u : u;                               // (-0 is 0)
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t) o << 32 | (uint32_t) ~token;
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t o = (uint32_t) (key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// e^d, d <= 0: off by a step of d's product with log2(e), which weighs little where d is far from 0
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896341f); }

// A lower bound of the wave's n-th largest key, at least n of which are not 0: bit by bit,
// counting the lanes that are not below. Sixteen bits do where no more than n more lanes are not
// below it, else all 64.
__device__ __forceinline__ uint64_t nth_largest(uint64_t key, uint32_t n) {
    const uint32_t hi = (uint32_t) (key >> 32), lo = (uint32_t) key;
    uint32_t t = 0, u = 0;
#pragma unroll
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) if ((uint32_t) __popcll(__ballot(hi >= (t | bit))) >= n) t |= bit;
    if ((uint32_t) __popcll(__ballot(hi >= t)) <= 2u * n) return (uint64_t) t << 32;
    for (uint32_t bit = 1u << 15; bit > 0; bit >>= 1) if ((uint32_t) __popcll(__ballot(hi >= (t | bit))) >= n) t |= bit;
    const uint32_t above = (uint32_t) __popcll(__ballot(hi > t));
    for (uint32_t bit = 1u << 31; bit > 0; bit >>= 1) if (above + (uint32_t) __popcll(__ballot(hi == t && lo >= (u | bit))) >= n) u |= bit;
    return (uint64_t) t << 32 | u;
}

// A wave's largest keys so far, a lane each, in falling order (0: none), of which the first n_pick
// count. A key is put in its place by one comparison in all lanes and a move of those behind it
// to the next lane.
struct wave_best {
    uint32_t hi, lo;                 // the lane's
    uint64_t least;                  // the n_pick-th
    uint32_t n_pick;

    __device__ __forceinline__ wave_best(uint32_t k) : hi(0), lo(0), least(0), n_pick(k) { }
    __device__ __forceinline__ uint64_t mine() const { return (uint64_t) hi << 32 | lo; }
    // the i-th, from 0 on
    __device__ __forceinline__ uint64_t place(uint32_t i) const {
        return (uint64_t) (uint32_t) __builtin_amdgcn_readlane((int) hi, (int) i) << 32 | (uint32_t) __builtin_amdgcn_readlane((int) lo, (int) i);
    }
    __device__ __forceinline__ void put_one(uint32_t h, uint32_t l) {        // (a key that is the same in all lanes)
        const uint64_t key = (uint64_t) h << 32 | l;
        // the lane in front's (wave_shr:1), the first lane's larger than all
        const uint32_t h1 = (uint32_t) __builtin_amdgcn_update_dpp(-1, (int) hi, 0x138, 0xf, 0xf, false);
        const uint32_t l1 = (uint32_t) __builtin_amdgcn_update_dpp(-1, (int) lo, 0x138, 0xf, 0xf, false);
        const bool stays = mine() > key, next = ((uint64_t) h1 << 32 | l1) > key;
        hi = stays ? hi : next ? h : h1;
        lo = stays ? lo : next ? l : l1;
    }
    // the keys of the lanes that take part
    __device__ __forceinline__ void put(bool take, uint64_t key) {
        for (uint64_t who = __ballot(take); who != 0; who &= who - 1) {
            const int at = __builtin_ctzll(who);
            put_one((uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) (key >> 32), at), (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) key, at));
        }
    }
    __device__ __forceinline__ void settle() {
        least = place(n_pick - 1);
    }
    // A first key of each lane (0: none), in order: a key's lane is how many are larger.
    __device__ __forceinline__ void start(uint64_t key) {
        const uint32_t h = (uint32_t) (key >> 32), l = (uint32_t) key;
        uint32_t rank = 0;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
            rank += ((uint64_t) (uint32_t) __builtin_amdgcn_readlane((int) h, i) << 32 | (uint32_t) __builtin_amdgcn_readlane((int) l, i)) > key;
        }
        // (those that are none all go behind the others; no lane's is none too)
        hi = (uint32_t) __builtin_amdgcn_ds_permute((int) (rank * 4u), (int) h);
        lo = (uint32_t) __builtin_amdgcn_ds_permute((int) (rank * 4u), (int) l);
        settle();
    }
    // What the keys of lanes with these largest ones have to reach to be among the first. Where
    // more lanes than picks have one above the list's last, the n_pick-th largest of them bounds the rest
    // from below, so that few are put in, in whatever order the values come.
    __device__ __forceinline__ uint64_t bound(uint64_t top) const {
        return (uint32_t) __popcll(__ballot(top > least)) > n_pick ? nth_largest(top, n_pick) : least + 1;
    }
};

// Rows of logits as a wave takes them: which lane takes which is counted from the row's start,
// so that a row's sums are the same bits wherever it lies. Rows of 16 bits that start within
// four bytes are loaded from the two bytes in front of them and moved over. Loads are bounded by
// the last whole four bytes of the row; a last two come by themselves.
template <typename T> struct beam_loads {
    static constexpr uint32_t PER = 16u / sizeof(T), N = BEAM_VALUES / PER;
    u32x4 v[N];
    uint32_t more[N];
    // where value i of a lane is, behind its first
    static __device__ __forceinline__ constexpr uint32_t token(uint32_t i) { return i / PER * 64u * PER + i % PER; }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, uint32_t at, bool odd) {
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) {
            const uint32_t by = (at + (j * 64u + (threadIdx.x & 63u)) * PER) * (uint32_t) sizeof(T);
            v[j] = __builtin_amdgcn_raw_buffer_load_b128(r, by, 0, 0);
            if (sizeof(T) == 2 && odd) more[j] = __builtin_amdgcn_raw_buffer_load_b32(r, by + 16u, 0, 0);
        }
    }
    __device__ __forceinline__ void values(float (&x)[BEAM_VALUES], bool odd) const {
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) {
            u32x4 w = v[j];
            if (sizeof(T) == 2 && odd) {
                w = (u32x4) { w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16 | more[j] << 16 };
            }
#pragma unroll
            for (uint32_t e = 0; e < PER; ++e) {
                if constexpr (sizeof(T) == 4) x[j * PER + e] = __uint_as_float(w[e]);
                else x[j * PER + e] = (float) __builtin_bit_cast(typename vec8<T>::type, w)[e];
            }
        }
    }
};

// A part of a row of logits: a reference at most 1 below the largest, the sum of exponentials
// relative to it, the best keys. Its waves take turns at 64 * BEAM_VALUES logits. Of their first ones they tell each other
// what n_pick keys of the part are no smaller than, and from then on put down what is not below that
// (128256 logits in four parts, 16 picks: about 100 of 32768), which is put in order at the end.
//
// 192 rows of 128256 bf16 logits, 49 MB, in 20.1 us, 2.5 TB/s; 15 without what is put down. Four rows of
// f32 5.7 us, of which a launch and a load from memory are most. Slower on the way here, us for the
// 192 rows: a list that all waves keep with barriers 64; a list a wave, ranked again for each tile 45;
// kept in order a key at a time 33, by bounds told after each tile 30; single values put down
// instead of a lane's eight 27. Logits that rise with the token cost twice as much, 47 in all for 256 rows.
template <typename T> __device__ __forceinline__ void beam_body(const att_beam_args &a) {
    typedef beam_loads<T> loads;
    // tiles of a wave that are on their way, 4 KB, and then gone through together
    constexpr uint32_t TILE = 64u * BEAM_VALUES, STEP = WAVES * TILE, AHEAD = sizeof(T) == 4 ? 2 : 4;
    typedef typename vec8<T>::type values;
    __shared__ values kept[WAVES][64u * (AHEAD + 1u)];
    __shared__ uint32_t kept_at[WAVES][64u * (AHEAD + 1u)];
    __shared__ uint64_t found[WAVES][128 + 8];
    __shared__ uint32_t n_found[WAVES];
    __shared__ float told[WAVES], part_m[WAVES];
    __shared__ double part_s[WAVES];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), row = blockIdx.x / a.n_chunk, c = blockIdx.x % a.n_chunk, end = a.n_vocab;
    if (a.ended && C_CAST(int32_t, a.ended)[row] >= 0) return;
    const float score = C_CAST(float, a.scores)[row];
    if (!(fabsf(score) <= -LOWEST)) return;
    const uint8_t *from = (const uint8_t *) a.logits + row * a.stride;
    const bool odd = sizeof(T) == 2 && ((uintptr_t) from & 2u) != 0;
    const uint32_t bytes = end * (uint32_t) sizeof(T) + (odd ? 2u : 0u);
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *) (from - (odd ? 2 : 0)), (short) 0, (int) uniform(bytes & ~3u), 0x00020000);
    const bool loose = (bytes & 3u) != 0;
    const uint32_t first = c * a.chunk + wave * TILE, last = min(c * a.chunk + a.chunk, end);
    loads ring[AHEAD];
#pragma unroll
    for (uint32_t u = 0; u < AHEAD; ++u) if (first + u * STEP < last) ring[u].load(r, first + u * STEP, odd);
    const float last_x = loose ? (float) G_CAST(const T, from)[end - 1] : 0.0f;
    wave_best best(a.n_pick);
    uint32_t n = 0, n_kept = 0;                                  // keys in `found`, lanes whose values are in `kept`
    float m = LOWEST, least = -INFINITY;                         // what is put down is not below `least`
    double sum = 0.0;
    // the waves with tiles, and which of a wave's largest it tells, from 0 on
    const uint32_t n_waves = min((uint32_t) WAVES, (last - c * a.chunk + TILE - 1u) / TILE), q = (a.n_pick - 1u) / n_waves;
    // what was found is put in order and given up, and what is below the last of n_pick is not found
    // again (what is alike may yet have a lower token: a lane's are not side by side)
    auto order = [&]() {
#pragma unroll 1
        for (uint32_t i = 0; i < n; i += 64u) {
            const uint64_t key = i + lane < n ? found[wave][i + lane] : 0;
            best.put(key >= best.bound(key), key);
            best.settle();
        }
        __builtin_amdgcn_wave_barrier();
        n = 0;
        if (best.least != 0) least = fmaxf(least, value_of(best.least));
    };
    // what was kept and is not below `least`, as keys: eight lanes' values at a time
    auto sift = [&]() {
#pragma unroll 1
        for (uint32_t i = 0; i < n_kept; i += 8u) {
            const uint32_t e = min(i + lane / BEAM_VALUES, n_kept - 1u), v = lane % BEAM_VALUES;
            const float x = (float) reinterpret_cast<const T *>(&kept[wave][e])[v];
            const uint32_t at = kept_at[wave][e] + loads::token(v);
            const bool take = i + lane / BEAM_VALUES < n_kept && x >= least && at < end;
            const uint64_t who = __ballot(take);
            if (take) found[wave][n + __builtin_amdgcn_mbcnt_hi((uint32_t) (who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t) who, 0))] = key_of(x, at);
            n += (uint32_t) __popcll(who);
            __builtin_amdgcn_wave_barrier();
            if (n > 64u) order();
        }
        n_kept = 0;
    };
    for (uint32_t t = first; t < last; t += AHEAD * STEP) {
        float x[AHEAD][BEAM_VALUES], top[AHEAD];
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u) {
            const uint32_t tu = t + u * STEP, tok = tu + lane * loads::PER;
            top[u] = -INFINITY;
            if (tu >= last) continue;
            ring[u].values(x[u], odd);
            if (tu + AHEAD * STEP < last) ring[u].load(r, tu + AHEAD * STEP, odd);
            if (tu + TILE > end) {
#pragma unroll
                for (uint32_t i = 0; i < BEAM_VALUES; ++i) {
                    const uint32_t at = tok + loads::token(i);
                    if (loose && at == end - 1) x[u][i] = last_x;
                    x[u][i] = at < end ? x[u][i] : -INFINITY;
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < BEAM_VALUES; ++i) top[u] = fmaxf(top[u], x[u][i]);  // (of NaN and a number, the number)
            if (top[u] > m + 1.0f) {                             // (else terms are at most e: rises that are small would add up their errors)
                sum *= (double) exp_of(m - top[u]);
                m = top[u];
            }
            float s = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < BEAM_VALUES; ++i) s += exp_of(x[u][i] - m);
            if (__any(s != s)) {                                 // NaN is -infinity
                s = 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < BEAM_VALUES; ++i) {
                    x[u][i] = fmaxf(x[u][i], -INFINITY);
                    s += exp_of(x[u][i] - m);
                }
            }
            sum += (double) s;
        }
        float most = top[0];
#pragma unroll
        for (uint32_t u = 1; u < AHEAD; ++u) most = fmaxf(most, top[u]);
        if (t == first) {                                        // (all waves with tiles are here)
            const uint64_t nth = (uint32_t) __popcll(__ballot(most > -INFINITY)) > q ? nth_largest(most > -INFINITY ? key_of(most, 0) : 0, q + 1u) : 0;
            if (lane == 0) told[wave] = nth == 0 ? -INFINITY : value_of(nth);
            __syncthreads();
            least = fminf(fminf(told[0], told[1]), fminf(told[2], told[3]));
        }
        // where more lanes than picks have something, as when logits rise with the token, these bound the rest
        if ((uint32_t) __popcll(__ballot(most >= least && most > -INFINITY)) > a.n_pick) {
            least = fmaxf(least, value_of(nth_largest(most > -INFINITY ? key_of(most, 0) : 0, a.n_pick)));
        }
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u) {
            const uint32_t tu = t + u * STEP, tok = tu + lane * loads::PER;
            const bool keep = top[u] >= least;
            const uint64_t who = __ballot(keep);
            if (tu >= last || who == 0) continue;
            if (keep) {                                          // (all its eight values: seldom more than one of them counts)
                const uint32_t e = n_kept + __builtin_amdgcn_mbcnt_hi((uint32_t) (who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t) who, 0));
                values y;                                        // (as they came)
#pragma unroll
                for (uint32_t i = 0; i < BEAM_VALUES; ++i) y[i] = (T) x[u][i];
                kept[wave][e] = y;
                kept_at[wave][e] = tok;
            }
            n_kept += (uint32_t) __popcll(who);
            __builtin_amdgcn_wave_barrier();
        }
        if (n_kept > 64u) {
            sift();
            // tokens rise from here on: what is alike the last comes behind it
            if (best.least != 0) least = fmaxf(least, value_of(((best.least >> 32) + 1u) << 32));
        }
    }
    if (first >= last) {                                         // (a wave without a tile)
        if (lane == 0) told[wave] = INFINITY;
        __syncthreads();
    }
    sift();
    if (__any(best.hi != 0)) {
        order();
        if (lane < a.n_pick) found[wave][lane] = best.mine();
        n = (uint32_t) __popcll(__ballot(lane < a.n_pick && best.hi != 0));
    }
    __builtin_amdgcn_wave_barrier();
    const uint64_t mine = lane < n ? found[wave][lane] : 0;
    if (lane < 8u) found[wave][n + lane] = 0;                    // (up to a multiple of eight)
    if (lane == 0) n_found[wave] = n;
    float all = m;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) all = fmaxf(all, __shfl_xor(all, d));
    if (lane == 0) part_m[wave] = all;
    __syncthreads();
    all = fmaxf(fmaxf(part_m[0], part_m[1]), fmaxf(part_m[2], part_m[3]));
    sum *= (double) exp_of(m - all);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) part_s[wave] = sum;
    // what the waves found, in order: a key's rank is how many are larger
    const uint64_t at = (uint64_t) row * a.n_chunk + c;
    uint32_t rank = 0, total = 0;
#pragma unroll 1
    for (uint32_t w = 0; w < WAVES; ++w) {
        const uint32_t nw = n_found[w];
        total += nw;
        for (uint32_t i = 0; i < nw; i += 8) {                   // (in eights: the reads do not wait for each other)
            uint64_t v[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) v[e] = found[w][i + e];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) rank += v[e] > mine;
        }
    }
    if (mine != 0 && rank < a.n_pick) G_CAST(uint64_t, a.keys)[at * a.n_pick + rank] = mine;
    if (tid >= total && tid < a.n_pick) G_CAST(uint64_t, a.keys)[at * a.n_pick + tid] = 0;
    __syncthreads();
    if (tid == 0) {
        G_CAST(double, a.sums)[2 * at] = (double) all;
        G_CAST(double, a.sums)[2 * at + 1] = part_s[0] + part_s[1] + part_s[2] + part_s[3];
    }
}

}  // namespace

#define BEAM(name, T) extern "C" __global__ void __launch_bounds__(ATT_THREADS) name(const att_beam_args a) { beam_body<T>(a); }
BEAM(sllm_k_beam_f32, float)
BEAM(sllm_k_beam_f16, _Float16)
BEAM(sllm_k_beam_bf16, __bf16)

// (4 beams of 63 parts 4.2 us, 32 groups of 8 beams of 4 parts 5.7: a launch, two loads that wait for each
// other, a logarithm in 64 bits.)
//
// A group: a wave joins a beam's parts (a lane a part, whose keys are in order: the largest of each, then
// the second, until none can be among the first), then its beams' lists are joined by their
// values in 64 bits. A beam that ended, or has no finite sum, is its token, and tokens from 0 on
// at -infinity.
extern "C" __global__ void __launch_bounds__(BEAM_JOIN_THREADS) sllm_k_beam_join(const att_beam_args a) {
    constexpr uint32_t AHEAD = 4;
    __shared__ double value[BEAM_MAX_LIST];
    __shared__ uint32_t token[BEAM_MAX_LIST];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), k = a.n_pick, row0 = blockIdx.x * a.n_beam;
    const uint32_t n_list = min(k, a.n_vocab);                   // of a beam
    for (uint32_t b = wave; b < a.n_beam; b += BEAM_JOIN_THREADS / 64) {
        const uint32_t row = row0 + b;
        // no more keys than lanes: one each; else each part's first ones. (Asked for before it is
        // known whether the beam has any.)
        const bool few = a.n_chunk * k <= 64u, in = lane < a.n_chunk;
        GLOBAL const double *sums = G_CAST(const double, a.sums) + 2 * ((uint64_t) row * a.n_chunk + lane);
        GLOBAL const uint64_t *keys = G_CAST(const uint64_t, a.keys) + ((uint64_t) row * a.n_chunk + lane) * k;
        uint64_t ahead[AHEAD];
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; ++j) ahead[j] = in && j < k && !few ? keys[j] : 0;
        if (few && lane < a.n_chunk * k) ahead[0] = G_CAST(const uint64_t, a.keys)[(uint64_t) row * a.n_chunk * k + lane];
        const double mine = in ? sums[0] : (double) LOWEST;
        double s = in ? sums[1] : 0.0;
        const float score = C_CAST(float, a.scores)[row];
        const int32_t end = a.ended ? C_CAST(int32_t, a.ended)[row] : -1;
        const bool fine = fabsf(score) <= -LOWEST;
        double m = (double) LOWEST, base = -INFINITY;
        if (fine && end < 0) {
            m = mine;
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) m = fmax(m, __shfl_xor(m, d));
            s *= exp(mine - m);
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
            base = (double) score - log(s);
            if (fabs(base) < INFINITY) {
                wave_best best(k);
                best.start(ahead[0]);
                for (uint32_t j = 0; j < k && !few; j += AHEAD) {
                    bool some = false;
#pragma unroll 1
                    for (uint32_t e = j == 0 ? 1u : 0u; e < AHEAD; ++e) {
                        const uint64_t one = e == 0 ? ahead[0] : e == 1 ? ahead[1] : e == 2 ? ahead[2] : ahead[3];
                        some = __any(one > best.least);
                        if (!some) break;
                        best.put(one >= best.bound(one), one);
                        best.settle();
                    }
                    if (!some) break;
#pragma unroll
                    for (uint32_t e = 0; e < AHEAD; ++e) ahead[e] = in && j + AHEAD + e < k ? keys[j + AHEAD + e] : 0;
                }
                if (lane < n_list) {
                    value[b * k + lane] = base + ((double) value_of(best.mine()) - m);
                    token[b * k + lane] = ~best.lo;
                }
                continue;
            }
        }
        if (lane < n_list) {
            const bool first = end >= 0 && fine;                 // its own token comes first
            uint32_t t = lane;
            if (first) t = lane == 0 ? (uint32_t) end : lane - 1 < (uint32_t) end ? lane - 1 : lane;
            value[b * k + lane] = first && lane == 0 ? (double) score : -INFINITY;
            token[b * k + lane] = t;
        }
    }
    __syncthreads();
    // a value's rank is its place and how many of each other beam's come first: of few values, the
    // beams are shared out among `per` threads of each
    const uint32_t n = a.n_beam * k;
    uint32_t per = 1;
    while (per < 64u && per < a.n_beam && 2u * per * n <= BEAM_JOIN_THREADS) per *= 2u;
    for (uint32_t i = tid / per; i < n; i += BEAM_JOIN_THREADS / per) {
        const uint32_t b = i / k, place = i % k;
        if (place >= n_list) continue;
        const double x = value[i];
        uint32_t rank = 0;
        for (uint32_t o = tid & (per - 1u); o < a.n_beam; o += per) {
            if (o == b) continue;
            uint32_t lo = 0;                                     // of a lower beam what is alike comes first too
            for (uint32_t hi = n_list; lo < hi;) {
                const uint32_t mid = (lo + hi) / 2;
                const double y = value[o * k + mid];
                if (y > x || (y == x && o < b)) lo = mid + 1;
                else hi = mid;
            }
            rank += lo;
        }
        for (uint32_t d = 1; d < per; d *= 2u) rank += __shfl_xor(rank, (int) d);
        rank += place;
        if ((tid & (per - 1u)) != 0) continue;
        if (rank >= k) continue;
        const uint64_t at = (uint64_t) blockIdx.x * k + rank;
        G_CAST(float, a.out)[at] = (float) x;
        G_CAST(int32_t, a.beam)[at] = (int32_t) b;
        G_CAST(int32_t, a.token)[at] = (int32_t) token[i];
    }
}
