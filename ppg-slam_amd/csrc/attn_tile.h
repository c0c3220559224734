// What the matrix-core attention kernels share: operand layouts, the running softmax, the two products of a tile.
//
// Scores are computed transposed, S^T = K Q^T, on v_mfma_f32_32x32x16 (16-bit types) or v_mfma_f32_32x32x2_f32: rows are 32
// keys, columns 32 queries.  A lane then holds 16 scores of ONE query (column lane & 31; the other 16 are in lane ^ 32), so
// maximum and sum need one exchange per tile, and the weights are already where the second product, O^T = V^T P^T, wants
// its B operand: sum over keys in the order that the lanes hold them.  For that V's operand is read in the same order, with
// the LDS read that transposes 16-bit numbers (four keys of one component per lane).
#pragma once
#include "attn_kernels.h"

namespace ppg {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// What a work-group needs to know of its set.
struct SetHere {
    int q0, nq, k0, nk, tile0, blk0, blocks;
};
__device__ __forceinline__ SetHere set_number(const AttnSets& sets, int s) {
    const int q0 = sets.q_off[s], k0 = sets.k_off[s], blk0 = sets.blk[s];
    return {q0, sets.q_off[s + 1] - q0, k0, sets.k_off[s + 1] - k0, sets.tile[s], blk0, sets.blk[s + 1] - blk0};
}
// What a launch has for all: its units, first and behind the last query row.  Asked for before any of it is looked at.
struct Launch {
    int units, q0, q1;
};
__device__ __forceinline__ Launch launch_of(const AttnSets& sets) {
    int units = sets.units, n = sets.n, q0 = sets.q_off[0];
    asm volatile("" : "+s"(units), "+s"(n), "+s"(q0));   // (the compiler would put the loads off)
    return {units, q0, sets.q_off[n]};
}
__device__ __forceinline__ Launch launch_of(const OneSet& set) { return {set.units, set.q0, set.q1}; }
// The set of tile, key block or query row x, the same for the wave; off ascends from off[0] <= x, INT_MAX behind the last set's end.
__device__ __forceinline__ int find_set(const int* off, int x, int lane) {
    static_assert(PPG_ATTN_MAX_SETS == 128, "two sets per lane");
    return __popcll(__ballot(off[lane + 1] <= x)) + __popcll(__ballot(off[lane + 65] <= x));
}
__device__ __forceinline__ SetHere set_of_tile(const AttnSets& sets, int x, int lane) { return set_number(sets, find_set(sets.tile, x, lane)); }
__device__ __forceinline__ SetHere set_of_block(const AttnSets& sets, int x, int lane) { return set_number(sets, find_set(sets.blk, x, lane)); }
__device__ __forceinline__ SetHere set_number(const OneSet& set, int) {
    int q0 = set.q0, q1 = set.q1, k0 = set.k0, k1 = set.k1, blocks = set.blocks;
    asm volatile("" : "+s"(q0), "+s"(q1), "+s"(k0), "+s"(k1), "+s"(blocks));
    return {q0, q1 - q0, k0, k1 - k0, 0, 0, blocks};
}
__device__ __forceinline__ SetHere set_of_tile(const OneSet& set, int, int) { return set_number(set, 0); }
__device__ __forceinline__ SetHere set_of_block(const OneSet& set, int, int) { return set_number(set, 0); }

// Bit r of m, and how many of its bits lie below the lane's, without a 64-bit shift by what a lane holds: with the amount in the last
// register of a wave's allocation such a shift has given wrong bits here (masks of a kernel that uses all 256).
struct Words {
    unsigned lo, hi;
};
__device__ __forceinline__ Words words_of(unsigned long long m) {   // m: the same for the wave
    unsigned lo = (unsigned)m, hi = (unsigned)(m >> 32);
    asm("" : "+s"(lo), "+s"(hi));   // (the compiler would make the two one 64-bit shift again)
    return {lo, hi};
}
__device__ __forceinline__ bool bit_of(Words m, int r) { return (((r & 32) ? m.hi : m.lo) >> (r & 31)) & 1; }
__device__ __forceinline__ int bits_below(unsigned long long m) { return __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0)); }

template <class T> struct IsF32 { static constexpr bool v = false; };
template <> struct IsF32<float> { static constexpr bool v = true; };

// 16-byte chunks: N components each, CPR per row of D; a lane's operand for 32 rows is NF of them
template <class T, int D> struct Shape {
    static constexpr int N = 16 / (int)sizeof(T), CPR = D / N, NF = CPR / 2;
    // chunk i of the operand of the lane half h: 16-bit: the 8 components that one MFMA wants from it; 32-bit: the two
    // halves of a row belong to the two lane halves (any pairing of components serves, the same for both operands)
    static __device__ __forceinline__ int chunk(int i, int h) { return IsF32<T>::v ? h * NF + i : 2 * i + h; }
    // LDS images keep a row's chunks permuted so that what one access touches lies in different banks (64 of them, 256 bytes):
    // the 16 rows of which 16 lanes take the same chunk, and the four rows by 64 bytes of a transposing read's 32 lanes
    static __device__ __forceinline__ int swz_k(int row) { return CPR >= 16 ? row & 15 : CPR == 8 ? (row >> 1) & 7 : (row >> 2) & 3; }
    static __device__ __forceinline__ int swz_v(int row) {
        if (IsF32<T>::v) return swz_k(row);
        return CPR >= 16 ? (row & 3) << 2 : CPR == 8 ? (row & 2) << 1 : 0;
    }
};

template <class T> __device__ __forceinline__ f32x16 mfma_chunk(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (IsF32<T>::v) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
        return c;
    } else if constexpr (__is_same(T, _Float16)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
}

// key of register r of a 32-key tile in the lane half h
__device__ __forceinline__ int key_of(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

__device__ __forceinline__ float other_half(float x, bool take_max) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float lo = __uint_as_float(r[0]), hi = __uint_as_float(r[1]);
    return take_max ? fmaxf(lo, hi) : lo + hi;
}

// how far a product may pass m before the sums are rescaled: 2^8 in the weights (finite also for the smallest scales, where no
// difference of products gets there)
__device__ __forceinline__ float rise_slack(float c) { return fminf(8.f / c, 3e38f); }

// Weights are 2^kLift times what the softmax says, in every sum alike: with fp16, whose smallest normal number is 2^-14, small ones
// then keep their precision (and the largest, 2^8 over m, are 2^15).
template <class T> constexpr float kLift = __is_same(T, _Float16) ? 7.f : 0.f;

// A weight's exponent is s c - m c, one instruction with m c computed once.  That m c is rounded: off by 2^-24 of itself, for all keys
// alike, but not alike for two stretches of keys with maxima of their own, and where it passes 2^31 or 32 bits themselves the weights
// under- or overflow altogether.  Beyond kFar (off by 2^-12 there) it is (s - m) c.  The test, once a tile, costs 1 % where the vector
// unit is the bound (64 streams: 101 -> 102 us); a flag set where m rises, and kept, cost up to 70 registers.
constexpr float kFar = 4096.f;

// Running softmax of the 32 queries of a wave, and their sums; m is the largest product seen (or up to 2^8 less in the
// exponent: the sums are rescaled only when a product passes it by that much, which any type holds), c = scale * log2 e.
//
// The sum of the weights: in l, added up by the vector unit, of this lane's half of the keys (the halves meet at the end); or
// (UNIT) in every component of u, by the matrix unit, as a product with ones.
template <class T, int D, bool UNIT = false> struct Running {
    using S = Shape<T, D>;
    f32x16 o[D / 32], u;
    float m, l;
    __device__ __forceinline__ float sum() const { return UNIT ? u[0] : other_half(l, false); }
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.f;
        if constexpr (UNIT)
#pragma unroll
            for (int r = 0; r < 16; r++) u[r] = 0.f;
#pragma unroll
        for (int t = 0; t < D / 32; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[t][r] = 0.f;
    }
    // largest score of this lane's query (both lane halves)
    template <int SUB> static __device__ __forceinline__ float largest(const f32x16 (&s)[SUB]) {
        float mt = s[0][0];
#pragma unroll
        for (int u = 0; u < SUB; u++)
#pragma unroll
            for (int r = 0; r < 16; r++) mt = fmaxf(mt, s[u][r]);
        return other_half(mt, true);
    }
    // makes room for scores up to mt
    __device__ __forceinline__ void rise(float mt, float c, float slack) {
        const bool up = mt - m > slack;   // (m + slack may round to more; -inf - -inf is no rise)
        if (__any(up)) {
            const float mn = up ? mt : m;
            const float alpha = mn == m ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c);
            m = mn;
            if constexpr (UNIT) {
#pragma unroll
                for (int r = 0; r < 16; r++) u[r] *= alpha;
            } else {
                l *= alpha;
            }
#pragma unroll
            for (int t = 0; t < D / 32; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[t][r] *= alpha;
        }
    }
    // weights in the place of the scores
    template <int SUB> __device__ __forceinline__ void weigh(f32x16 (&s)[SUB], float c) {
        float mc = (m == -INFINITY ? 0.f : m * c) - kLift<T>;   // (nothing so far: every weight below is exp2(-inf))
        float sum[2] = {0.f, 0.f};
        const bool far = fabsf(mc) > kFar;
        if (__any(far)) {   // (in place, and nothing for queries that are not: their weights do not depend on which others are in the wave)
            const float by = far ? m : 0.f;
            mc = far ? -kLift<T> : mc;
#pragma unroll
            for (int u = 0; u < SUB; u++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[u][r] -= by;
        }
#pragma unroll
        for (int u = 0; u < SUB; u++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], c, -mc));
                if constexpr (!UNIT) sum[r & 1] += s[u][r];
            }
        if constexpr (!UNIT) l += sum[0] + sum[1];
    }
    template <int SUB> __device__ __forceinline__ void weights(f32x16 (&s)[SUB], float c, float slack) {
        rise(largest(s), c, slack);
        weigh(s, c);
    }
};

// o += P V of 32 keys; v: LDS image of the values, key0 the keys' first row in it.  The weights are rounded to the values' type
// here, once.
template <class T, int D, bool UNIT>
__device__ __forceinline__ void add_values(Running<T, D, UNIT>& run, const f32x16& p, const char* v, int key0, int lane) {
    using S = Shape<T, D>;
    const int h = lane >> 5;
    if constexpr (IsF32<T>::v) {
        static_assert(!UNIT, "the 32-bit matrix unit is the bottleneck: sums are the vector unit's");
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int row = key0 + key_of(r, h);
#pragma unroll
            for (int t = 0; t < D / 32; t++) {
                const int d = t * 32 + (lane & 31);
                const float a = *(const float*)(v + row * (D * 4) + ((((d >> 2) ^ S::swz_v(row)) << 4) | ((d & 3) << 2)));
                run.o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], run.o[t], 0, 0, 0);
            }
        }
    } else {
        const int i = lane & 15, part = (lane >> 4) & 1;
#pragma unroll
        for (int st = 0; st < 2; st++) {
            T pb[8];
#pragma unroll
            for (int e = 0; e < 8; e++) pb[e] = (T)p[8 * st + e];
            const u32x4 b = __builtin_bit_cast(u32x4, pb);
            if constexpr (UNIT) {
                const short one = __builtin_bit_cast(short, (T)1.f);
                const s16x8 ones = {one, one, one, one, one, one, one, one};
                run.u = mfma_chunk<T>(__builtin_bit_cast(u32x4, ones), b, run.u);
            }
            const int r0 = key0 + 16 * st + 4 * h + (i >> 2), r1 = r0 + 8;
#pragma unroll
            for (int t = 0; t < D / 32; t++) {
                const int ch = t * 4 + part * 2 + ((i & 3) >> 1), in = (i & 1) * 8;
                const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(v + r0 * (D * 2) + ((ch ^ S::swz_v(r0)) << 4) + in));
                const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(v + r1 * (D * 2) + ((ch ^ S::swz_v(r1)) << 4) + in));
                const s16x8 a = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
                run.o[t] = mfma_chunk<T>(__builtin_bit_cast(u32x4, a), b, run.o[t]);
            }
        }
    }
}

// Scores of masked keys (bit set in `dead`, the same for the wave; bit 0 = the tile's first key) become -inf, whatever the product
// gave.  Eight keys at a time, four of each lane half: with few keys masked most groups cost a scalar test.
__device__ __forceinline__ void mask_scores(f32x16& s, unsigned dead, int h) {
#pragma unroll
    for (int b = 0; b < 4; b++) {
        if (!((dead >> (8 * b)) & 0xff)) continue;
        const int d = (int)((dead >> (8 * b)) >> (4 * h));
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const unsigned x = (unsigned)((d << (31 - e)) >> 31);   // all ones where masked
            s[4 * b + e] = __uint_as_float(__builtin_amdgcn_bitop3_b32(x, 0xff800000u, __float_as_uint(s[4 * b + e]), 0xca));   // x ? -inf : s
        }
    }
}

// Divisions are long chains of dependent instructions in a work-group's start.  24 bits (numbers of work-groups, heads, parts) have a
// short one, which the compiler takes when it sees that there are no more.
__device__ __forceinline__ int quot24(int a, int b) { return (int)(((unsigned)a & 0xffffff) / ((unsigned)b & 0xffffff)); }
__device__ __forceinline__ int rem24(int a, int b) { return (int)(((unsigned)a & 0xffffff) % ((unsigned)b & 0xffffff)); }
// where share i of n things begins, of `shares` equal ones
__device__ __forceinline__ int share_begin(int n, int i, int shares) {
    if (shares == 1) return i ? n : 0;
    const unsigned each = (unsigned)n / (unsigned)shares, more = (unsigned)n - each * (unsigned)shares;
    return (int)(each * (unsigned)i + min((unsigned)i, more));
}

// work-group L of a launch of n units: XCD L % 8 (launch order) serves a contiguous range of the units, so that the units that
// read the same keys meet in one L2; n or more: nothing to do
__device__ __forceinline__ int xcd_unit(int L, int n) {
    const int per = (n + 7) >> 3;
    const int u = (L & 7) * per + (L >> 3);
    return (L >> 3) < per ? u : n;
}
__host__ __device__ inline unsigned xcd_grid(int n) { return 8u * (unsigned)((n + 7) >> 3); }

}  // namespace ppg
