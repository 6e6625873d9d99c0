// attn_kernels.hip -- attention over a paged cache and over packed prompts, and
// the cache's copies (sllm_gfx950_attn.h), for gfx950.
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
// has rows of its own and all share a tile. PAGED: keys are found by page.
template <typename A, typename T, int D, int NT, bool KEYS, bool PAGED>
struct attention {
    typedef tile<T, D, KEYS> L;
    static constexpr bool WIDE = L::WIDE;
    static constexpr bool SPLIT = !WIDE && sizeof(A) == 4;       // f32 rows against f16 keys
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

    __device__ __forceinline__ void places() {
        const uint32_t row = a.hd * (uint32_t) sizeof(T);
        const uint32_t rowk = PAGED ? row : (uint32_t) a.k_tok, rowv = PAGED ? row : (uint32_t) a.v_tok;
#pragma unroll
        for (int q = 0; q < QC; ++q) {
            if (!KEYS) koff[q] = li * L::ROWB + (((4u * q + g) ^ L::ksw(li)) * 16u);
            else kcopy[q] = (4u * q + g) * 16u < row ? li * rowk + (4u * q + g) * 16u : PAST;
        }
        const uint32_t r = WIDE ? 4u * g : 4u * g + (li >> 2);
        voff = L::VALUES + r * L::ROWB + (WIDE ? ((li >> 2) ^ L::vsw(r)) * 16u + (li & 3u) * 4u
                                             : (((li >> 1) & 1u) ^ L::vsw(r)) * 16u + (li & 1u) * 8u);
#pragma unroll
        for (int j = 0; j < COPIES; ++j) {
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
    t8 qf[WIDE ? 1 : NT][WIDE ? 1 : QC], ql[SPLIT ? NT : 1][SPLIT ? QC : 1];
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
            } else if constexpr (!SPLIT) {
#pragma unroll
                for (int s = 0; s < QC; ++s) {
                    const uint32_t d = 8u * (4u * s + g);
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
    struct span { const uint8_t *k, *v; };
    __device__ __forceinline__ span rows_at(uint32_t key) const {
        if constexpr (PAGED) {
            const uint32_t at = min(key, it.key1 - 1u);
            const uint32_t page = *C_CAST(uint32_t, a.tables + it.kv + (at >> a.page_shift));
            const uint64_t off = page * a.page_bytes + ((uint64_t) (it.head << a.page_shift) + (at & ((1u << a.page_shift) - 1u) & ~(uint32_t) (GROUP - 1))) * (a.hd * (uint32_t) sizeof(T));
            return { a.k + off, a.v + off };
        } else {
            return { a.k + (uint64_t) (it.kv + key) * a.k_tok + it.head * a.k_head, a.v + (uint64_t) (it.kv + key) * a.v_tok + it.head * a.v_head };
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
        // a sequence's own keys are read once and not kept (2: nontemporal): 64.9 -> 60.6 us
        // for 8 sequences of 16384 positions, bf16; a prompt's are read by many workgroups
        constexpr int KEPT = PAGED ? 2 : 0;
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
        t8 p[WIDE ? 1 : NT], rest[SPLIT ? NT : 1];
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
                    if constexpr (WIDE) sum += x;
                    if constexpr (WIDE) {
                        p.w[nt][i] = x;
                    } else {
                        p.p[nt][4 * ks + i] = (T) x;
                        if constexpr (SPLIT) p.rest[nt][4 * ks + i] = (T) (x - (float) p.p[nt][4 * ks + i]);
                    }
                }
            }
            if constexpr (!WIDE) {
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
                    if constexpr (SPLIT) o[dt][nt] = mfma(vf, p.rest[nt], o[dt][nt]);
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
        if constexpr (KEYS) {
            fetch(x, spans(t), t);
        } else {
            issue(t, stage(0));
            issue(t + 1, stage(1));
        }
    }

    // KEYS: tile t, in registers, which then take the next (two tiles on their way at a
    // time were no faster: 58.8 us and 57.4 for 8 sequences of 16384 positions, bf16)
    template <bool CAREFUL>
    __device__ __forceinline__ void turn(uint32_t t) {
        const uint32_t then = t + STEP;
        const span_of_tile m = spans(then);                      // (past the end: the last page again)
        scores s;
        clear(s);
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
    // vector instructions each: within 2 % of each other.)
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

    // The same with care, a tile after the other.
    __device__ __forceinline__ void careful_pass() {
        begin();
        if (it.key0 >= it.key1) return;
        const uint32_t t1 = (it.key1 + KT - 1u) / KT;
        for (uint32_t t = first_tile(); t < t1; t += STEP) {
            if constexpr (KEYS) {
                fetch(x, spans(t), t);
                turn<true>(t);
            } else {
                issue(t, stage(0));
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

template <typename A, typename T, int D, int NT, bool KEYS, bool PAGED>
__device__ __forceinline__ void attend_item(const att_args &a, const att_item &it, uint8_t *S) {
    const uint32_t lane = threadIdx.x & 63u;
    attention<A, T, D, NT, KEYS, PAGED> x = { a, it, S, lane, uniform(threadIdx.x >> 6), lane >> 4, lane & 15u };
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

}  // namespace

#define PROMPT(name, T, D) extern "C" __global__ void __launch_bounds__(ATT_THREADS, 2) name(const att_args a) { prompt_body<T, D>(a); }
#define PAGED(name, A, T, D) extern "C" __global__ void __launch_bounds__(ATT_THREADS, 2) name(const att_args a) { paged_body<A, T, D>(a); }

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

// Pages to pages: blockIdx.y a pair of them, ATT_COPY_CHUNKS 16-byte pieces of
// what it holds a workgroup, all four of a thread's in flight together. Bound by
// memory: 396 pages of 655 KB moved or copied in two launches 92 us, 5.5 TB/s; 16 copies
// of 41 positions of 30 layers, a source that the caches hold, 15.2 us, 3.5 TB/s.
extern "C" __global__ void __launch_bounds__(ATT_THREADS) sllm_k_attn_copy(const att_copy_args a) {
    const att_pair p = a.pair[blockIdx.y];
    const uint32_t per = p.rows * a.row_bytes / 16u, n = per * a.n_blocks;
    const uint8_t *src = a.mem + p.src * a.page_bytes;
    uint8_t *dst = a.mem + p.dst * a.page_bytes;
    constexpr int UN = ATT_COPY_CHUNKS / ATT_THREADS;
    u32x4 v[UN];
    uint64_t at[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
        const uint32_t x = blockIdx.x * ATT_COPY_CHUNKS + (uint32_t) i * ATT_THREADS + threadIdx.x;
        at[i] = (uint64_t) (x / per) * a.block_bytes + (x % per) * 16u;
        if (x < n) v[i] = *G_CAST(const u32x4, src + at[i]);
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
        const uint32_t x = blockIdx.x * ATT_COPY_CHUNKS + (uint32_t) i * ATT_THREADS + threadIdx.x;
        if (x < n) *G_CAST(u32x4, dst + at[i]) = v[i];
    }
}
