// Attention on the matrix cores, over whole sets or over selected blocks (layouts and softmax in attn_tile.h).
//
// Rows: the queries of the `group` heads that share a key head are one long list, row r = query r / group, head r % group.
//   attention_wide_kernel  four waves of 32 rows each share the key and value tiles in LDS (two stages: the next tile's
//                          loads are in flight in registers while this one is multiplied);
//   attention_split_kernel 32 rows per work-group, its four waves (and, where rows are few, several work-groups) share out the
//                          keys; sums meet in LDS, and those of several work-groups in attention_join_kernel.
// Selected blocks, few queries: attention_split_kernel too, the listed blocks of ONE query as its keys.
// Selected blocks, many queries: the lists are turned round (bin_kernel: for every block the queries that name it), so that a
// block's keys and values are read once for all of them (attention_blocks_kernel, a wave per block and 32 rows), and every
// (query, place in its list) leaves its sums for attention_join_kernel.
#include "attn_tile.h"

#include <algorithm>
#include <type_traits>

namespace ppg {

// where row r of key head g lives; rows behind the last are the last one (computed, not stored)
struct RowPlace {
    long long q;
    int head;
};
__device__ __forceinline__ RowPlace row_place(int r, int rows, int group, int g, int q0) {
    r = min(r, rows - 1);
    const int q = group == 1 ? r : r / group;
    return {(long long)(q0 + q), g * group + (group == 1 ? 0 : r - q * group)};
}

template <class T, int D, int NF = Shape<T, D>::NF>
__device__ __forceinline__ void load_query(u32x4 (&f)[NF], const ppg_rows& q, const RowPlace& p, int h) {
    const T* x = (const T*)q.p + p.q * q.row + p.head * q.head;
#pragma unroll
    for (int i = 0; i < Shape<T, D>::NF; i++) f[i] = *(const u32x4*)(x + Shape<T, D>::chunk(i, h) * Shape<T, D>::N);
}

// The same for a wave's 32 rows by way of an LDS image of its own, when its lanes know their rows' addresses (`mine`: of row
// lane & 31): neighbouring lanes then load a row's neighbouring chunks, where a lane per row touches 32 or 64 lines with every load
// (a frame pair's work-groups spent a quarter of their time on that).
template <class T, int D, int NF = Shape<T, D>::NF> __device__ __forceinline__ void fetch_rows(u32x4 (&x)[NF], const T* mine, int lane) {
    using S = Shape<T, D>;
    const unsigned long long at = (unsigned long long)mine;
#pragma unroll
    for (int i = 0; i < S::NF; i++) {
        const int c = lane + 64 * i, r = c / S::CPR;
        const T* y = (const T*)(((unsigned long long)(unsigned)__shfl((int)(at >> 32), r) << 32) | (unsigned)__shfl((int)at, r));
        x[i] = *(const u32x4*)(y + (c % S::CPR) * S::N);
    }
}
template <class T, int D, int NF = Shape<T, D>::NF> __device__ __forceinline__ void rows_to_operand(u32x4 (&f)[NF], const u32x4 (&x)[NF], char* image, int lane) {
    using S = Shape<T, D>;
    constexpr int ROWB = D * (int)sizeof(T);
    const int row = lane & 31, h = lane >> 5;
#pragma unroll
    for (int i = 0; i < S::NF; i++) {
        const int c = lane + 64 * i, r = c / S::CPR;
        *(u32x4*)(image + r * ROWB + (((c % S::CPR) ^ S::swz_k(r)) << 4)) = x[i];
    }
    __builtin_amdgcn_wave_barrier();   // (LDS serves a wave in order)
#pragma unroll
    for (int i = 0; i < S::NF; i++) f[i] = *(const u32x4*)(image + row * ROWB + ((S::chunk(i, h) ^ S::swz_k(row)) << 4));
    __builtin_amdgcn_wave_barrier();
}

// Rows of 32-bit results: this lane's components of its own row, 4 consecutive ones per register group.
template <int D> __device__ __forceinline__ void store_row(float* y, const f32x16 (&o)[D / 32], float f, int h) {
#pragma unroll
    for (int t = 0; t < D / 32; t++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            f32x4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = f == 0.f ? 0.f : o[t][b * 4 + e] * f;
            *(f32x4*)(y + t * 32 + 8 * b + 4 * h) = w;
        }
}
// Rows of 16-bit results (E), by way of an LDS image of the wave's own (32 rows of D): a row is then stored by neighbouring
// lanes, 16 bytes each, in one piece.  f: factor of this lane's row; to(r): where row r goes, or null.
template <class E, int D, class To> __device__ __forceinline__ void store_rows(char* image, const f32x16 (&o)[D / 32], float f, int lane, To to) {
    constexpr int CPR = D / 8;
    const int h = lane >> 5, row = lane & 31;
    auto place = [&](int r, int ch) { return image + r * (D * 2) + ((ch ^ (r & (CPR - 1))) << 4); };
#pragma unroll
    for (int t = 0; t < D / 32; t++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            E w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = (E)(f == 0.f ? 0.f : o[t][b * 4 + e] * f);
            *(s16x4*)(place(row, t * 4 + b) + 8 * h) = __builtin_bit_cast(s16x4, w);
        }
    __builtin_amdgcn_wave_barrier();   // (LDS serves a wave in order)
#pragma unroll
    for (int i = 0; i < 32 * CPR / 64; i++) {
        const int r = (lane + 64 * i) / CPR, ch = (lane + 64 * i) % CPR;
        E* y = (E*)to(r);
        const u32x4 v = *(const u32x4*)place(r, ch);
        if (y) *(u32x4*)(y + ch * 8) = v;
    }
}
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : 1.f / l; }
template <class T> __device__ __forceinline__ float log_sum(float m, float l, float scale) { return l == 0.f ? -INFINITY : fmaf(m, scale, (__log2f(l) - kLift<T>) * kLn2); }

// Sums of every (row, part) between two kernels: D components each, so that they lie in whole lines (lists of 8 streams: 181 us, 198 with m and l
// behind each vector), and behind all of them (m, l).  A part without keys has m = -inf, l = 0.
template <int D> struct Parts {
    float* o;
    float2* ml;
    __device__ __forceinline__ Parts(void* work, const Launch& here, int heads, int parts)
        : o((float*)work), ml((float2*)(o + (long long)(here.q1 - here.q0) * heads * parts * D)) {}
};
inline size_t parts_bytes(long long n, int head_dim) { return (size_t)n * (head_dim + 2) * sizeof(float); }

// Four waves of 32 rows each.  8192 x 8191 keys, 2 heads of 128, 4 sets: 303 us, 907 TFLOP/s, where a library product of 8192^3
// reaches 1122; 64 streams of about 870, 4 heads of 64: 102 us, 490 TFLOP/s (with 8192 keys a set: 810).  Counters at 64
// components: the vector unit (exponentials, maxima, conversions: 155 instructions for 64 keys) is busy for 61 % of the time,
// the matrix unit for 47 %, at 2.0 GHz, the clock that the power limit leaves; what short sets lose is the work-group's start
// (queries, first tiles) and the chip's last round.  Two waves of a SIMD in opposite phases, held there by barriers, measured
// slower (315 and 1555 us instead of 303 and 1367): a single wave cannot keep the vector unit busy.
// 32-bit types (the matrix unit reaches 154 TFLOP/s): 64 components 124 TFLOP/s (4 sets of 4096 a side, 4 heads; 64 sets of 870: 103),
// 32 components 115, 128 components 103 (84 for short sets): there two waves a SIMD spill 38 registers, some inside the loop.
// parts > 1: a work-group takes its share of the keys and leaves its sums.
// Which keys are masked is read once, a bit each, kWindow words ahead, so that the loads of a tile do not wait for it.
// UNIT (16-bit types): the matrix unit adds up the weights (a product with ones); the vector unit, which has the exponentials, is
// the busier one (4 % of the time at 64 and at 128 components).  Those are the rounded weights, the same that meet the
// values, but their sum is not good enough for a log: with lse the vector unit adds up the unrounded ones.
constexpr int kWindow = 64;   // 64-key words of the mask in LDS at a time
template <class T, int D, int BN, bool UNIT, class Sets>
__global__ __launch_bounds__(256, D == 128 || (IsF32<T>::v && D == 64) ? 2 : 3) void attention_wide_kernel(AttentionLaunch a, Sets sets, int parts) {
    using S = Shape<T, D>;
    constexpr int SUB = BN / 32, CH = BN * S::CPR / 256, ROWB = D * (int)sizeof(T), TILE = BN * ROWB, STEP = 256 / S::CPR;
    constexpr unsigned long long FULL = BN == 64 ? ~0ull : 0xffffffffull;
    static_assert(BN * S::CPR % 256 == 0, "tile loads are whole rounds of the work-group");
    __shared__ alignas(16) char lds_k[2][TILE], lds_v[2][TILE];
    __shared__ unsigned long long lds_dead[kWindow];
    const Launch here = launch_of(sets);
    const int units = here.units * parts, whole = xcd_unit(blockIdx.x, units);
    if (whole >= units) return;
    const int unit = parts == 1 ? whole : quot24(whole, parts), part = parts == 1 ? 0 : rem24(whole, parts);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const SetHere set = set_of_tile(sets, unit, lane);
    const int q0 = set.q0, k0 = set.k0, nk = set.nk, kvh = a.k.heads, group = quot24(a.q.heads, kvh);
    const int rows = set.nq * group, tiles = (rows + 127) / 128;
    const int g = quot24(unit - set.tile0, tiles), row = rem24(unit - set.tile0, tiles) * 128 + wave * 32 + (lane & 31);
    const float c = a.scale * kLog2e, slack = rise_slack(c);
    const int all = (nk + BN - 1) / BN, from = share_begin(all, part, parts), to = share_begin(all, part + 1, parts);

    // tile loads: thread -> (row, chunk) and STEP rows on
    const int r0 = tid / S::CPR, ch0 = tid % S::CPR;
    const T* kp = (const T*)a.k.p + g * a.k.head + (long long)k0 * a.k.row + ch0 * S::N;
    const T* vp = (const T*)a.v.p + g * a.v.head + (long long)k0 * a.v.row + ch0 * S::N;
    const T *kr = kp + r0 * a.k.row, *vr = vp + r0 * a.v.row;
    u32x4 rk[CH], rv[CH];
    auto fetch = [&](int t) {
        const long long j = (long long)t * BN;
        if (j + BN <= nk) {   // the same for all
            const T *x = kr + j * a.k.row, *y = vr + j * a.v.row;
#pragma unroll
            for (int i = 0; i < CH; i++) {
                rk[i] = *(const u32x4*)(x + (long long)STEP * i * a.k.row);
                rv[i] = *(const u32x4*)(y + (long long)STEP * i * a.v.row);
            }
        } else {   // rows behind the set are its last one
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const long long r = min(j + r0 + STEP * i, (long long)nk - 1);
                rk[i] = *(const u32x4*)(kp + r * a.k.row);
                rv[i] = *(const u32x4*)(vp + r * a.v.row);
            }
        }
    };
    auto store = [&](int t, unsigned long long dead) {   // masked values are zero
        const Words w = words_of(dead);
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const int r = r0 + STEP * i;
            const unsigned live = bit_of(w, r) ? 0u : ~0u;
            *(u32x4*)(lds_k[t & 1] + r * ROWB + ((ch0 ^ S::swz_k(r)) << 4)) = rk[i];
            *(u32x4*)(lds_v[t & 1] + r * ROWB + ((ch0 ^ S::swz_v(r)) << 4)) = rv[i] & u32x4{live, live, live, live};
        }
    };
    // the places of a tile that hold no key to attend to
    auto window = [&](int t) {   // of the kWindow words from tile t's on
        for (int w = wave; w < kWindow; w += 4) {
            const long long j = (long long)t * BN + w * 64 + lane;
            if (j - lane >= min((long long)nk, (long long)to * BN)) break;
            const unsigned long long m = __ballot(j >= nk || a.skip[k0 + (int)min(j, (long long)nk - 1)] != 0);
            if (lane == 0) lds_dead[w] = m;
        }
    };
    auto dead_of = [&](int t) -> unsigned long long {
        unsigned long long m;
        if (a.skip) {
            const int i = t - from;
            const unsigned long long x = lds_dead[(i * (BN / 32) / 2) % kWindow] >> (BN == 32 ? (i & 1) * 32 : 0);
            m = ((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)x);
        } else {
            const long long left = nk - (long long)t * BN;
            m = left >= BN ? 0 : ~0ull << left;
        }
        return m & FULL;
    };
    constexpr int PER_WINDOW = kWindow * 64 / BN;   // tiles

    unsigned long long dead = 0;   // of the tile being multiplied
    const RowPlace place = row_place(row, rows, group, g, q0);
    u32x4 qf[S::NF];
    load_query<T, D>(qf, a.q, place, h);
    Running<T, D, UNIT> run;
    run.clear();
    if (from < to) {
        fetch(from);
        if (a.skip) {
            window(from);
            __syncthreads();
        }
        dead = dead_of(from);
        store(from, dead);
    }
    __syncthreads();
    for (int t = from; t < to; t++) {
        const int buf = t & 1;
        unsigned long long next = 0;
        if (t + 1 < to) {
            if (a.skip && (t + 1 - from) % PER_WINDOW == 0) {   // (all words so far have been read, before the last barrier)
                window(t + 1);
                __syncthreads();
            }
            next = dead_of(t + 1);
            fetch(t + 1);
        }
        f32x16 sc[SUB];
        __builtin_amdgcn_s_setprio(1);   // the matrix unit's share first: 4 % at 128 components, nothing at 64
#pragma unroll
        for (int u = 0; u < SUB; u++) {
            const int r = u * 32 + (lane & 31);
#pragma unroll
            for (int e = 0; e < 16; e++) sc[u][e] = 0.f;
#pragma unroll
            for (int i = 0; i < S::NF; i++) {
                const u32x4 kf = *(const u32x4*)(lds_k[buf] + r * ROWB + ((S::chunk(i, h) ^ S::swz_k(r)) << 4));
                sc[u] = mfma_chunk<T>(kf, qf[i], sc[u]);
            }
            if (dead) mask_scores(sc[u], (unsigned)(dead >> (32 * u)), h);
        }
        __builtin_amdgcn_s_setprio(0);
        run.template weights<SUB>(sc, c, slack);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int u = 0; u < SUB; u++) add_values(run, sc[u], lds_v[buf], u * 32, lane);
        __builtin_amdgcn_s_setprio(0);
        if (t + 1 < to) store(t + 1, next);   // last read one tile ago, before the barrier below
        dead = next;
        __syncthreads();
    }
    const float l = run.sum();
    if (parts > 1) {
        if (row >= rows) return;
        const Parts<D> to(a.work, here, a.q.heads, parts);
        const long long at = (long long)((int)(place.q - here.q0) * a.q.heads + place.head) * parts + part;
        store_row<D>(to.o + at * D, run.o, 1.f, h);
        if (h == 0) to.ml[at] = make_float2(run.m, l);
        return;
    }
    if (a.lse && h == 0 && row < rows) a.lse[place.q * a.q.heads + place.head] = log_sum<T>(run.m, l, a.scale);
    if constexpr (IsF32<T>::v) {
        if (row < rows) store_row<D>((float*)a.out.p + place.q * a.out.row + place.head * a.out.head, run.o, inverse_sum(l), h);
    } else {
        static_assert(2 * TILE >= 128 * ROWB, "the key tiles' place holds the rows (their last reads are behind the last barrier)");
        const int first = row - (lane & 31);
        store_rows<T, D>(lds_k[0] + wave * 32 * ROWB, run.o, inverse_sum(l), lane, [&](int r) -> void* {
            if (first + r >= rows) return nullptr;
            const RowPlace p = row_place(first + r, rows, group, g, q0);
            return (T*)a.out.p + p.q * a.out.row + p.head * a.out.head;
        });
    }
}

// A wave's own stretch of keys: keys, then values, through an LDS image of its own.
// One row against 400003 keys, 4 heads of 64: 410 MB in 79 us, 5.2 TB/s (a copy reaches 5.1, half of it written; with a
// lane per row for the keys' loads, 85 us).
template <class T, int D, int BN> struct OwnKeys {
    using S = Shape<T, D>;
    static constexpr int SUB = BN / 32, VC = BN * S::CPR / 64, ROWB = D * (int)sizeof(T);
    u32x4 rk[VC], rv[VC];
    int masked;                  // this lane's key of the tile (the first BN lanes)
    unsigned long long gone;     // all of them, once settle() was called
    const T *kp, *vp;            // the set's first key and value, the same for the wave
    const uint8_t* skip;
    long long k_row, v_row;
    unsigned k_at, v_at;         // this lane's place in a round of loads, in bytes, if it is `near` enough for 32 bits
    bool near;
    static constexpr int STEP = 64 / S::CPR;   // rows of a round
    __device__ __forceinline__ void begin(const T* k, const T* v, long long k_row_, long long v_row_, const uint8_t* skip_, int lane) {
        kp = k;
        vp = v;
        skip = skip_;
        k_row = k_row_;
        v_row = v_row_;
        near = (k_row | v_row) < (1 << 24);
        k_at = lane / S::CPR * (unsigned)k_row * sizeof(T) + lane % S::CPR * 16;
        v_at = lane / S::CPR * (unsigned)v_row * sizeof(T) + lane % S::CPR * 16;
    }
    // keys first + j0 .. first + j0 + BN - 1, of which those below first + n exist (n >= 1: row n - 1 stands in for those behind it)
    __device__ __forceinline__ void load(int first, int j0, int n, int lane) {
        const int j = j0 + (lane & (BN - 1));
        masked = skip ? skip[first + min(j, n - 1)] : 0;   // first: loads come back in order, and this one is waited for first
        if (j >= n) masked = 1;
        if (near && j0 + BN <= n) {   // the same for the wave; addresses are its own, but for one offset per lane
            const char *x = (const char*)(kp + (long long)(first + j0) * k_row), *y = (const char*)(vp + (long long)(first + j0) * v_row);
#pragma unroll
            for (int i = 0; i < VC; i++) rk[i] = *(const u32x4*)(x + (long long)(STEP * i * sizeof(T)) * k_row + k_at);
#pragma unroll
            for (int i = 0; i < VC; i++) rv[i] = *(const u32x4*)(y + (long long)(STEP * i * sizeof(T)) * v_row + v_at);
        } else {
#pragma unroll
            for (int i = 0; i < VC; i++) {
                const int x = lane + 64 * i, r = x / S::CPR;
                rk[i] = *(const u32x4*)(kp + (long long)(first + min(j0 + r, n - 1)) * k_row + (x % S::CPR) * S::N);
            }
#pragma unroll
            for (int i = 0; i < VC; i++) {
                const int x = lane + 64 * i, r = x / S::CPR;
                rv[i] = *(const u32x4*)(vp + (long long)(first + min(j0 + r, n - 1)) * v_row + (x % S::CPR) * S::N);
            }
        }
    }
    __device__ __forceinline__ void settle(int lane) { gone = __ballot(lane < BN && masked); }
    __device__ __forceinline__ void values_to_lds(char* v, int lane) const {
        const Words w = words_of(gone);
#pragma unroll
        for (int i = 0; i < VC; i++) {
            const int x = lane + 64 * i, r = x / S::CPR, ch = x % S::CPR;
            *(u32x4*)(v + r * ROWB + ((ch ^ S::swz_v(r)) << 4)) = bit_of(w, r) ? u32x4{0, 0, 0, 0} : rv[i];
        }
    }
    __device__ __forceinline__ void scores(f32x16 (&sc)[SUB], const u32x4 (&qf)[S::NF], char* image, int lane) const {
        const int h = lane >> 5;
#pragma unroll
        for (int i = 0; i < VC; i++) {
            const int x = lane + 64 * i, r = x / S::CPR, ch = x % S::CPR;
            *(u32x4*)(image + r * ROWB + ((ch ^ S::swz_k(r)) << 4)) = rk[i];
        }
        __builtin_amdgcn_wave_barrier();   // the image is this wave's own and LDS serves a wave in order
#pragma unroll
        for (int u = 0; u < SUB; u++) {
            const int r = u * 32 + (lane & 31);
#pragma unroll
            for (int e = 0; e < 16; e++) sc[u][e] = 0.f;
#pragma unroll
            for (int i = 0; i < S::NF; i++) {
                const u32x4 kf = *(const u32x4*)(image + r * ROWB + ((S::chunk(i, h) ^ S::swz_k(r)) << 4));
                sc[u] = mfma_chunk<T>(kf, qf[i], sc[u]);
            }
            if (gone) mask_scores(sc[u], (unsigned)(gone >> (32 * u)), h);
        }
        __builtin_amdgcn_wave_barrier();
    }
};

// The sums of the four waves of a work-group meet in LDS; who stores a row's components adds them up, from wave 0 upwards.
template <int D> struct Meeting {
    float o[4][32][D + 4];   // + 4: the 32 rows that a 16-byte access takes start in different banks
    float m[4][32], l[4][32];
};
template <class T, int D> __device__ __forceinline__ void to_meeting(Meeting<D>& x, const Running<T, D>& run, int wave, int lane) {
    const int h = lane >> 5, col = lane & 31;
    store_row<D>(x.o[wave][col], run.o, 1.f, h);
    const float l = run.sum();
    if (h == 0) {
        x.m[wave][col] = run.m;
        x.l[wave][col] = l;
    }
}
// components d .. d + 3 of row r, its m and l
template <int D> __device__ __forceinline__ f32x4 of_meeting(const Meeting<D>& x, int r, int d, float c, float& m, float& l) {
    m = fmaxf(fmaxf(x.m[0][r], x.m[1][r]), fmaxf(x.m[2][r], x.m[3][r]));
    l = 0.f;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const float f = x.m[w][r] == m ? 1.f : __builtin_amdgcn_exp2f((x.m[w][r] - m) * c);
        l += x.l[w][r] * f;
        y += *(const f32x4*)&x.o[w][r][d] * f;
    }
    return y;
}

// SEL: a unit's rows are the group of one query, its keys the blocks of that query's list.
template <class T, int D, int BN, bool SEL, class Sets>
__global__ __launch_bounds__(256, IsF32<T>::v && D == 128 ? 1 : 2) void attention_split_kernel(AttentionLaunch a, Sets sets, int parts) {
    using S = Shape<T, D>;
    constexpr int SUB = BN / 32, IMG = BN * D * (int)sizeof(T);
    __shared__ alignas(16) union {
        char v[4][IMG];
        Meeting<D> sums;
    } lds;
    const Launch here = launch_of(sets);
    const int units = here.units * parts, unit = xcd_unit(blockIdx.x, units);
    if (unit >= units) return;
    const int part = rem24(unit, parts), tile = quot24(unit, parts);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const SetHere set = set_of_tile(sets, tile, lane);
    const int q0 = set.q0, k0 = set.k0, nk = set.nk, kvh = a.k.heads, group = quot24(a.q.heads, kvh);
    // SEL: tiles of a query's group never hold rows of another query
    const int nq = set.nq, all = nq * group, per_q = (group + 31) / 32, tiles = SEL ? nq * per_q : (all + 31) / 32;
    const int g = quot24(tile - set.tile0, tiles), at = rem24(tile - set.tile0, tiles);
    const int row0 = SEL ? at / per_q * group + at % per_q * 32 : at * 32;
    const int rows = SEL ? (at / per_q + 1) * group : all;
    const RowPlace place = row_place(row0 + (lane & 31), rows, group, g, q0);
    u32x4 qx[S::NF], qf[S::NF];
    fetch_rows<T, D>(qx, (const T*)a.q.p + place.q * a.q.row + place.head * a.q.head, lane);
    const float c = a.scale * kLog2e, slack = rise_slack(c);
    Running<T, D> run;
    run.clear();
    const T* kp = (const T*)a.k.p + g * a.k.head + (long long)k0 * a.k.row;
    const T* vp = (const T*)a.v.p + g * a.v.head + (long long)k0 * a.v.row;
    const int* sel = SEL ? a.sel + ((long long)(q0 + at / per_q) * kvh + g) * a.n_sel : nullptr;
    const int per_shift = SEL && a.block > BN ? __builtin_ctz((unsigned)a.block / BN) : 0, blocks = SEL ? (nk + a.block - 1) / a.block : 0;
    // SEL: a lane per place of the list, and those that name a block moved to the front; the waves take their tiles in turn.
    // Whole sets: a stretch for every part, whose tiles the waves take in turn.
    int listed = -1, named = 0;
    if constexpr (SEL) {
        static_assert(PPG_ATTN_MAX_SEL <= 64, "a lane per place");
        listed = lane < a.n_sel ? sel[lane] : -1;
        const unsigned long long ok = __ballot(listed >= 0 && listed < blocks);
        named = __popcll(ok);
        const int before = bits_below(ok), place = listed >= 0 && listed < blocks ? before : named + lane - before;
        listed = __builtin_amdgcn_ds_permute(place << 2, listed);
    }
    const int nt = SEL ? named << per_shift : (int)(((unsigned)nk + BN - 1) / BN);
    const int from = SEL ? part * 4 : share_begin(nt, part, parts), to = SEL ? nt : share_begin(nt, part + 1, parts), stride = SEL ? 4 * parts : 4;
    OwnKeys<T, D, BN> keys;
    keys.begin(kp, vp, a.k.row, a.v.row, a.skip ? a.skip + k0 : nullptr, lane);
    auto load = [&](int t) {
        if constexpr (SEL) {
            const int first = __builtin_amdgcn_readlane(listed, t >> per_shift) * a.block, j = (t & ((1 << per_shift) - 1)) * BN;
            keys.load(first, j, min(a.block, nk - first), lane);
        } else {
            keys.load(0, t * BN, nk, lane);
        }
    };
    if (from + wave < to) load(from + wave);
    rows_to_operand<T, D>(qf, qx, lds.v[wave], lane);
    for (int t = from + wave; t < to; t += stride) {
        f32x16 sc[SUB];
        keys.settle(lane);
        keys.scores(sc, qf, lds.v[wave], lane);
        keys.values_to_lds(lds.v[wave], lane);
        if (t + stride < to) load(t + stride);
        run.template weights<SUB>(sc, c, slack);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < SUB; u++) add_values(run, sc[u], lds.v[wave], u * 32, lane);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    to_meeting(lds.sums, run, wave, lane);
    __syncthreads();
    // 32 rows x D components out, 4 per thread and round
    for (int i = threadIdx.x; i < 32 * (D / 4); i += 256) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4;
        if (row0 + r >= rows) continue;
        float m, l;
        const f32x4 y = of_meeting(lds.sums, r, d, c, m, l);
        const RowPlace p = row_place(row0 + r, rows, group, g, q0);
        if (parts > 1) {
            const Parts<D> to(a.work, here, a.q.heads, parts);
            const long long at = (long long)((int)(p.q - here.q0) * a.q.heads + p.head) * parts + part;
            *(f32x4*)(to.o + at * D + d) = y;
            if (d == 0) to.ml[at] = make_float2(m, l);
            continue;
        }
        const float inv = inverse_sum(l);
        T out[4];
#pragma unroll
        for (int e = 0; e < 4; e++) out[e] = (T)(inv == 0.f ? 0.f : y[e] * inv);
        T* to_ = (T*)a.out.p + p.q * a.out.row + p.head * a.out.head + d;
        if constexpr (IsF32<T>::v) *(f32x4*)to_ = __builtin_bit_cast(f32x4, out);
        else *(s16x4*)to_ = __builtin_bit_cast(s16x4, out);
        if (a.lse && d == 0) a.lse[p.q * a.q.heads + p.head] = log_sum<T>(m, l, a.scale);
    }
}

// Joins the parts of every (row, head): a team's threads take 16 bytes of components each, PG such teams the parts of one
// (row, head) in turn, four loads in flight; the teams' sums meet in LDS in their order.  SEL: part i belongs to place i of the
// query's list and exists only if that names a block.
template <int D> struct JoinShape {
    static constexpr int C = 4, TEAM = D / C, TEAMS = 256 / TEAM;
};
template <class T, int D, bool SEL, int PG, class Sets>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionLaunch a, Sets sets, int parts) {
    using J = JoinShape<D>;
    constexpr int C = J::C, TEAM = J::TEAM, TEAMS = J::TEAMS;
    typedef float vec __attribute__((ext_vector_type(C)));
    struct Sum {
        vec o;
        float m, l;
    };
    __shared__ Sum met[PG > 1 ? 256 : 1];
    const int team = threadIdx.x / TEAM, sub = team % PG, d = threadIdx.x % TEAM * C;
    const Launch here = launch_of(sets);
    const unsigned heads = a.q.heads, n = (unsigned)(here.q1 - here.q0) * heads, at = blockIdx.x * (TEAMS / PG) + team / PG;
    const unsigned rh = min(at, n - 1);   // (a team behind the last does its work again and keeps it to itself)
    const float c = a.scale * kLog2e;
    const Parts<D> all(a.work, here, a.q.heads, parts);
    const float* w = all.o + (long long)rh * parts * D + d;
    const float2* ml = all.ml + (long long)rh * parts;
    const long long q = here.q0 + (int)(rh / heads);
    const int head = (int)(rh % heads);
    int blocks = 0;
    const int* sel = nullptr;
    if constexpr (SEL) {
        if constexpr (__is_same(Sets, OneSet)) {
            blocks = sets.blocks;
        } else {   // the set of the work-group's first row, and on from there
            const unsigned first = min(blockIdx.x * (TEAMS / PG), n - 1);
            int s = find_set(sets.q_off, here.q0 + (int)(first / heads), threadIdx.x & 63);
            while (q >= sets.q_off[s + 1]) s++;
            blocks = sets.blk[s + 1] - sets.blk[s];
        }
        sel = a.sel + (q * a.k.heads + head / (a.q.heads / a.k.heads)) * a.n_sel;
    }
    float m = -INFINITY, l = 0.f;
    vec o = {};
    for (int p0 = sub; p0 < parts; p0 += 4 * PG) {
        Sum x[4];
        bool on[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int p = min(p0 + i * PG, parts - 1);
            x[i].m = ml[p].x;
            x[i].l = ml[p].y;
            x[i].o = *(const vec*)(w + p * D);
            on[i] = p0 + i * PG < parts;
            if constexpr (SEL) on[i] = on[i] && (unsigned)sel[p] < (unsigned)blocks;
        }
        float mn = m;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (on[i]) mn = fmaxf(mn, x[i].m);
        const float keep = m == mn ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c);
        m = mn;
        l *= keep;
        o *= keep;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (on[i]) {
                const float f = x[i].m == m ? 1.f : __builtin_amdgcn_exp2f((x[i].m - m) * c);
                l += x[i].l * f;
                o += x[i].o * f;
            }
    }
    if constexpr (PG > 1) {
        met[threadIdx.x] = Sum{o, m, l};
        __syncthreads();
        if (sub) return;
        for (int i = 1; i < PG; i++) {
            const Sum x = met[threadIdx.x + i * TEAM];
            const float mn = fmaxf(m, x.m), keep = m == mn ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c), add = x.m == mn ? 1.f : __builtin_amdgcn_exp2f((x.m - mn) * c);
            m = mn;
            l = l * keep + x.l * add;
            o = o * keep + x.o * add;
        }
    }
    if (at >= n) return;
    const float inv = inverse_sum(l);
    struct alignas(C * sizeof(T)) Out { T v[C]; } out;
#pragma unroll
    for (int e = 0; e < C; e++) out.v[e] = (T)(inv == 0.f ? 0.f : o[e] * inv);
    *(Out*)((T*)a.out.p + q * a.out.row + head * a.out.head + d) = out;
    if (a.lse && d == 0) a.lse[q * a.q.heads + head] = log_sum<T>(m, l, a.scale);
}

// ---- selected blocks, many queries ----
// A region is one (set, key head); its entries are the places in the lists of its queries.  Where things lie:
struct BinWork {
    unsigned* list;   // entries by block, [regions][queries of the set * n_sel]: query of the set << entry_shift | place
    int4* tile;       // (block, its first entry in the list, first of the tile's rows among entries * group, set << 22 | key head << 6 | rows of the tile); block -1: unused
};
__host__ __device__ inline int entry_shift(int n_sel) { return n_sel > 1 ? 32 - __builtin_clz((unsigned)n_sel - 1) : 0; }   // (queries * n_sel < 2^30)
static_assert(PPG_ATTN_MAX_SETS <= 128, "seven bits for the set");
// A region's blocks are counted by one work-group, or in kBinShares equal shares by as many where the entries are more than the
// blocks (region_tiles() then has room for every block's last tile) and every share has blocks (what a share without any would
// have to know, the entries before it, it does not count).
constexpr int kBinShares = 4;
__host__ __device__ inline int bin_shares(long long nq, int n_sel, int blocks) {
    return nq * n_sel >= 2048 && nq * n_sel >= blocks && blocks >= 4 * kBinShares ? kBinShares : 1;
}
// tiles that a region may need: its rows in 32s, and one more for every block's last
__host__ __device__ inline int region_tiles(long long nq, int n_sel, int group, int blocks) {
    const long long e = nq * n_sel;
    return (int)(e * group / 32 + (e < blocks ? e : blocks));
}

// One work-group per share of a region's blocks: counts per block, their running sum, and the entries put in their places.  Which
// entry of a block comes first is left to the atomics: entries of a block never meet in a sum.  A share's entries start
// behind those of the blocks before it (every share counts them), its tiles where those blocks' could end at the latest.
// (The form for one set spills 26 registers, the other none.  One frame of 500 queries x 16: 9 us from 16 work-groups; 8 streams: 13 us.)
constexpr int kBins = 8192;    // blocks counted at a time (32 KB of LDS)
constexpr int kBinHold = 16;   // entries per thread that stay in registers between the two passes
template <class Sets>
__global__ __launch_bounds__(1024) void bin_kernel(AttentionLaunch a, Sets sets, BinWork w) {
    __shared__ int cnt[kBins];
    __shared__ int sum_e[16], sum_t[16], sum_b[16];
    const int kvh = a.k.heads, group = quot24(a.q.heads, kvh), s = quot24(blockIdx.x, kvh), g = rem24(blockIdx.x, kvh);
    const Launch here = launch_of(sets);
    const SetHere set = set_number(sets, s);
    const int q0 = set.q0, nq = set.nq, blocks = set.blocks, n = nq * a.n_sel;
    const int* sel = a.sel + ((long long)q0 * kvh + g) * a.n_sel;
    const int step = kvh * a.n_sel, shift = entry_shift(a.n_sel);
    const int list0 = ((q0 - here.q0) * kvh + g * nq) * a.n_sel;   // of this region's entries
    unsigned* list = w.list + list0;
    int4* tile = w.tile + set.tile0 + (long long)g * region_tiles(nq, a.n_sel, group, blocks);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int shares = bin_shares(nq, a.n_sel, blocks), share = blockIdx.y;
    if (share >= shares) return;
    const int lo = share_begin(blocks, share, shares), hi = share_begin(blocks, share + 1, shares);
    int e0 = 0, t0 = 0;   // where the entries and tiles of this round's bins go
    int held[kBinHold], rank[kBinHold];
    const bool once = n <= kBinHold * 1024;
    const int dq = 1024 / a.n_sel, dr = 1024 % a.n_sel;   // 1024 entries on, in queries and places
    // this thread's entries of the kBinHold * 1024 from `from` on (one at a time: neighbouring lanes take neighbouring entries, which
    // name different blocks; four at a time 4 us more for 8 streams): f(which, query, place)
    auto each = [&](int from, auto f) {
        int q = (from + tid) / a.n_sel, r = (from + tid) % a.n_sel;
#pragma unroll
        for (int i = 0; i < kBinHold; i++) {
            if (from + i * 1024 >= n) break;   // the same for all
            f(i, q, r);
            q += dq;
            r += dr;
            if (r >= a.n_sel) {
                r -= a.n_sel;
                q++;
            }
        }
    };
    auto load = [&](int from) {
#pragma unroll
        for (int i = 0; i < kBinHold; i++) held[i] = -1;
        each(from, [&](int i, int q, int r) {
            if (from + i * 1024 + tid < n) held[i] = sel[q * step + r];
        });
    };
    for (int b0 = lo; b0 < hi; b0 += kBins) {
        const int nb = min(kBins, hi - b0), per = (nb + 1023) / 1024;
        for (int i = tid; i < nb; i += 1024) cnt[i] = 0;
        int below = 0;
        if (b0 == lo) load(0);
        __syncthreads();
        for (int from = 0; from < n; from += kBinHold * 1024) {
            if (!once) load(from);
#pragma unroll
            for (int i = 0; i < kBinHold; i++) {
                if (from + i * 1024 >= n) break;
                if (held[i] >= b0 && held[i] - b0 < nb) rank[i] = atomicAdd(&cnt[held[i] - b0], 1);
                below += held[i] >= 0 && held[i] < lo;
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) below += __shfl_xor(below, d);
        if (lane == 0) sum_b[wave] = below;
        __syncthreads();
        if (b0 == lo) {
            for (int i = 0; i < 16; i++) e0 += sum_b[i];
            if (lo) t0 = (int)((long long)e0 * group / 32) + lo;
        }
        int es = 0, ts = 0;
        for (int i = tid * per; i < min(nb, (tid + 1) * per); i++) {
            es += cnt[i];
            ts += (cnt[i] * group + 31) / 32;
        }
        int ei = es, ti = ts;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(ei, d), y = __shfl_up(ti, d);
            if (lane >= d) {
                ei += x;
                ti += y;
            }
        }
        if (lane == 63) {
            sum_e[wave] = ei;
            sum_t[wave] = ti;
        }
        __syncthreads();
        int eb = e0 + ei - es, tb = t0 + ti - ts;
        for (int i = 0; i < 16; i++) {
            if (i < wave) {
                eb += sum_e[i];
                tb += sum_t[i];
            }
            e0 += sum_e[i];
            t0 += sum_t[i];
        }
        for (int i = tid * per; i < min(nb, (tid + 1) * per); i++) {
            const int c = cnt[i], rows = c * group;
            for (int r = 0; r < rows; r += 32) tile[tb++] = make_int4(b0 + i, list0 + eb, r, s << 22 | g << 6 | min(32, rows - r));
            cnt[i] = eb;   // where the block's next entry goes
            eb += c;
        }
        __syncthreads();
        for (int from = 0; from < n; from += kBinHold * 1024) {
            if (!once) load(from);
            each(from, [&](int i, int q, int r) {
                const int b = held[i];
                if (b >= b0 && b - b0 < nb) list[once ? cnt[b - b0] + rank[i] : atomicAdd(&cnt[b - b0], 1)] = (unsigned)q << shift | r;
            });
        }
        __syncthreads();
    }
    // up to where the next share's tiles start
    const int end = share + 1 < shares ? (int)((long long)e0 * group / 32) + hi : region_tiles(nq, a.n_sel, group, blocks);
    for (int i = t0 + tid; i < end; i += 1024) tile[i] = make_int4(-1, 0, 0, 0);
}

// Bound by memory: 8 streams of 1024 rows, 16 of 1025 blocks of 64 keys each, 4 heads of 64: 547 MB of inputs and results and 277 MB of
// parts, written and read, in 181 us for the three kernels (13 turning the lists, 134 here, 33 joining).  (Parts in fp16 were 20 us less, and lost what is left where the blocks'
// values cancel.)
// A wave per tile: one block's keys against 32 rows out of the queries that name it.  32 keys at a time: fewer registers, so that
// three waves of a SIMD have loads in flight (64 at a time: 15 us more for 8 streams; two waves sharing a block: 10 % more).
template <class T, int D, class Sets>
__global__ __launch_bounds__(64, IsF32<T>::v && D == 128 ? 1 : 2) void attention_blocks_kernel(AttentionLaunch a, Sets sets, BinWork w) {
    using S = Shape<T, D>;
    constexpr int BN = 32, SUB = BN / 32, IMG = BN * D * (int)sizeof(T);
    __shared__ alignas(16) char lds_v[IMG];
    const int lane = threadIdx.x, h = lane >> 5;
    // (in launch order: hardly two tiles read the same block, and a region's unused tiles would leave some XCDs without work)
    const int4 t = w.tile[blockIdx.x];
    const Launch here = launch_of(sets);
    const int block = __builtin_amdgcn_readfirstlane(t.x), region = __builtin_amdgcn_readfirstlane(t.w);
    if (block < 0) return;
    const SetHere set = set_number(sets, region >> 22);
    const int g = (region >> 6) & 0xffff, left = region & 63;   // (1..32 rows)
    const int group = quot24(a.q.heads, a.k.heads), rr = t.z + min(lane & 31, left - 1);
    const int in = group == 1 ? rr : rr / group;
    const unsigned entry = w.list[t.y + in];   // before the keys, which are not waited for so soon
    const int first = block * a.block, n = min(a.block, set.nk - first);
    OwnKeys<T, D, BN> keys;
    keys.begin((const T*)a.k.p + g * a.k.head + (long long)set.k0 * a.k.row, (const T*)a.v.p + g * a.v.head + (long long)set.k0 * a.v.row, a.k.row,
               a.v.row, a.skip ? a.skip + set.k0 : nullptr, lane);
    keys.load(first, 0, n, lane);
    const int shift = entry_shift(a.n_sel), slot = entry & ((1u << shift) - 1), head = g * group + (group == 1 ? 0 : rr - in * group);
    const long long q = set.q0 + (int)(entry >> shift);
    u32x4 qx[S::NF], qf[S::NF];
    fetch_rows<T, D>(qx, (const T*)a.q.p + q * a.q.row + head * a.q.head, lane);
    rows_to_operand<T, D>(qf, qx, lds_v, lane);
    const float c = a.scale * kLog2e, slack = rise_slack(c);
    Running<T, D> run;
    run.clear();
    for (int j = 0; j < n; j += BN) {
        f32x16 sc[SUB];
        keys.settle(lane);
        keys.scores(sc, qf, lds_v, lane);
        keys.values_to_lds(lds_v, lane);
        if (j + BN < n) keys.load(first, j + BN, n, lane);
        run.template weights<SUB>(sc, c, slack);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < SUB; u++) add_values(run, sc[u], lds_v, u * 32, lane);
        __builtin_amdgcn_wave_barrier();
    }
    const float l = run.sum();
    if ((lane & 31) >= left) return;   // (both lane halves of a row leave together)
    const Parts<D> to(a.work, here, a.q.heads, a.n_sel);
    const int at = ((int)(q - here.q0) * a.q.heads + head) * a.n_sel + slot;
    store_row<D>(to.o + (long long)at * D, run.o, 1.f, h);
    if (h == 0) to.ml[at] = make_float2(run.m, l);
}

// ---- which kernel ----
namespace {

struct DensePlan {
    bool wide;
    int parts;
};
constexpr int kFill = 512;   // work-groups that fill the chip (two per CU)

// units of `rows` rows of the call into sets.tile
int count_tiles(const AttentionLaunch& a, AttnSets& sets, int rows) {
    const long long kvh = a.k.heads, group = a.q.heads / kvh;
    sets.tile[0] = 0;
    for (int s = 0; s < sets.n; s++)
        sets.tile[s + 1] = sets.tile[s] + (int)(((sets.q_off[s + 1] - (long long)sets.q_off[s]) * group + rows - 1) / rows * kvh);
    return end_tiles(sets);
}
DensePlan dense_plan(int dtype, int head_dim, const AttentionLaunch& a, AttnSets& sets) {
    const bool f32 = dtype == PPG_F32;
    long long longest = 0;
    for (int s = 0; s < sets.n; s++) longest = std::max(longest, (long long)sets.k_off[s + 1] - sets.k_off[s]);
    const int few = count_tiles(a, sets, 32), many = count_tiles(a, sets, 128);
    if (many >= kFill) return {true, 1};
    // More than 32 rows: their keys are worth sharing, if that still gives half the chip work of four tiles each (117 queries x 4
    // heads of 128 on one key head against 219142 keys: 96 us, 280 us in 32s; 40 queries x 4 heads of 64 against 100000: 33 and 41).
    const int wide_most = (int)std::min<long long>(longest / (4 * (f32 ? 32 : 64)), kFill);
    if (many && few >= 2 * many && many * wide_most >= kFill / 2) return {true, std::min(wide_most, kFill / many)};
    count_tiles(a, sets, 32);
    const int bn = f32 || head_dim == 128 ? 32 : 64;
    // a part has a tile for each of its waves; no more parts than run at once
    const long long most = std::max(1LL, (longest + 4 * bn - 1) / (4 * bn));
    return {false, few ? (int)std::min<long long>(most, std::max(1, kFill / few)) : 1};
}

// selected blocks
struct BlocksPlan {
    bool binned;
    int parts;
    size_t part_bytes, list_bytes, tile_bytes;   // of the binned form, in this order
};
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
// A query's blocks are read for itself, in one launch instead of three, while that is no more than this many bytes of keys and
// values.  16 of 313 blocks, 4 heads, direct against turned round in us, at 64 MB and where the second overtakes: 64 keys x 64
// components bf16 11.6 : 16.8, 175 MB; x 128 14.6 : 18.4, 150 MB; x 32 10.6 : 16.4, 125 MB; fp32 x 64 19.4 : 25.3, 95 MB; x 128
// 30.6 : 34.1, 75 MB; 32 keys x 64 bf16 14.0 : 16.5, 75 MB: below it for all of these.
constexpr long long kDirectBytes = 64LL << 20;
BlocksPlan blocks_plan(int dtype, int head_dim, const AttentionLaunch& a, AttnSets& sets) {
    const long long nq = (long long)sets.q_off[sets.n] - sets.q_off[0], kvh = a.k.heads, group = a.q.heads / kvh;
    BlocksPlan p{};
    sets.tile[0] = 0;
    long long named = 0, longest = 1;   // (query, block)s at most, and of one query
    for (int s = 0; s < sets.n; s++) {
        const long long most = std::max(1, std::min(a.n_sel, sets.blk[s + 1] - sets.blk[s]));
        named += (sets.q_off[s + 1] - (long long)sets.q_off[s]) * most;
        longest = std::max(longest, most);
    }
    if (named * kvh * a.block * head_dim * (dtype == PPG_F32 ? 8 : 4) > kDirectBytes) {
        p.binned = true;
        p.parts = a.n_sel;
        for (int s = 0; s < sets.n; s++)
            sets.tile[s + 1] = sets.tile[s] + (int)kvh * region_tiles(sets.q_off[s + 1] - sets.q_off[s], a.n_sel, (int)group, sets.blk[s + 1] - sets.blk[s]);
        end_tiles(sets);
        end_list(sets, sets.q_off);
        p.part_bytes = up256(parts_bytes(nq * a.q.heads * a.n_sel, head_dim));
        p.list_bytes = up256((size_t)nq * kvh * a.n_sel * sizeof(int));
        p.tile_bytes = up256((size_t)sets.units * sizeof(int4));
        return p;
    }
    const long long per_q = (group + 31) / 32;
    for (int s = 0; s < sets.n; s++) sets.tile[s + 1] = sets.tile[s] + (int)((sets.q_off[s + 1] - sets.q_off[s]) * per_q * kvh);
    const int units = end_tiles(sets), bn = dtype == PPG_F32 || head_dim == 128 ? 32 : 64;
    const long long most = std::max(1LL, (longest * ((a.block + bn - 1) / bn) + 3) / 4);
    p.parts = units ? (int)std::min<long long>(most, std::max(1, kFill / units)) : 1;
    if (p.parts > 1) p.part_bytes = parts_bytes(nq * a.q.heads * p.parts, head_dim);
    return p;
}

template <class T, int D, bool SEL> hipError_t join(const AttentionLaunch& a, AttnSets& sets, int parts, hipStream_t s) {
    using J = JoinShape<D>;
    constexpr int TEAMS = J::TEAMS, MANY = std::min(16, TEAMS);
    const long long n = ((long long)sets.q_off[sets.n] - sets.q_off[0]) * a.q.heads;
    // one team per (row, head) where those fill the chip, else several
    const int pg = n * J::TEAM >= 65536 * 2 || parts < 8 ? 1 : parts < 32 ? 4 : MANY;
    const unsigned grid = (unsigned)((n + TEAMS / pg - 1) / (TEAMS / pg));
    auto go = [&](const auto& st) {
        using Sets = std::decay_t<decltype(st)>;
        if (pg == 1) attention_join_kernel<T, D, SEL, 1, Sets><<<grid, 256, 0, s>>>(a, st, parts);
        else if (pg == 4) attention_join_kernel<T, D, SEL, 4, Sets><<<grid, 256, 0, s>>>(a, st, parts);
        else attention_join_kernel<T, D, SEL, MANY, Sets><<<grid, 256, 0, s>>>(a, st, parts);
        return hipGetLastError();
    };
    if constexpr (SEL) return with_sets(sets, go);
    else return go(OneSet(sets));
}
template <class T, int D> hipError_t run(const AttentionLaunch& a, AttnSets& sets, int dtype, hipStream_t s) {
    constexpr int WIDE_BN = IsF32<T>::v ? 32 : 64, OWN_BN = IsF32<T>::v || D == 128 ? 32 : 64;
    hipError_t e;
    auto split = [&](auto sel, int parts) {
        return with_sets(sets, [&](const auto& st) {
            attention_split_kernel<T, D, OWN_BN, decltype(sel)::value, std::decay_t<decltype(st)>><<<xcd_grid(sets.units * parts), 256, 0, s>>>(a, st, parts);
            return hipGetLastError();
        });
    };
    if (a.sel) {
        const BlocksPlan p = blocks_plan(dtype, D, a, sets);
        if (!sets.units && !p.binned) return hipSuccess;
        if (!p.binned) {
            e = split(std::true_type(), p.parts);
            return e != hipSuccess || p.parts == 1 ? e : join<T, D, false>(a, sets, p.parts, s);
        }
        BinWork w;
        w.list = (unsigned*)((char*)a.work + p.part_bytes);
        w.tile = (int4*)((char*)w.list + p.list_bytes);
        if (sets.units) {
            e = with_sets(sets, [&](const auto& st) {
                using Sets = std::decay_t<decltype(st)>;
                bin_kernel<Sets><<<dim3(sets.n * a.k.heads, kBinShares), 1024, 0, s>>>(a, st, w);
                const hipError_t first = hipGetLastError();
                if (first != hipSuccess) return first;
                attention_blocks_kernel<T, D, Sets><<<(unsigned)sets.units, 64, 0, s>>>(a, st, w);
                return hipGetLastError();
            });
            if (e != hipSuccess) return e;
        }
        return join<T, D, true>(a, sets, p.parts, s);
    }
    const DensePlan p = dense_plan(dtype, D, a, sets);
    if (!sets.units) return hipSuccess;
    if (p.wide) {
        const unsigned grid = xcd_grid(sets.units * p.parts);
        e = with_sets(sets, [&](const auto& st) {
            using Sets = std::decay_t<decltype(st)>;
            if (a.lse || IsF32<T>::v) attention_wide_kernel<T, D, WIDE_BN, false, Sets><<<grid, 256, 0, s>>>(a, st, p.parts);
            else attention_wide_kernel<T, D, WIDE_BN, !IsF32<T>::v, Sets><<<grid, 256, 0, s>>>(a, st, p.parts);
            return hipGetLastError();
        });
        return e != hipSuccess || p.parts == 1 ? e : join<T, D, false>(a, sets, p.parts, s);
    }
    e = split(std::false_type(), p.parts);
    return e != hipSuccess || p.parts == 1 ? e : join<T, D, false>(a, sets, p.parts, s);
}
template <class T> hipError_t run_dim(const AttentionLaunch& a, AttnSets& sets, int dtype, int head_dim, hipStream_t s) {
    return head_dim == 32 ? run<T, 32>(a, sets, dtype, s) : head_dim == 64 ? run<T, 64>(a, sets, dtype, s) : run<T, 128>(a, sets, dtype, s);
}

}  // namespace

size_t attention_work(int dtype, int head_dim, const AttentionLaunch& a, AttnSets& sets) {
    if (a.n_sel) {
        const BlocksPlan p = blocks_plan(dtype, head_dim, a, sets);
        // (a list's sums are joined by head_dim / 4 threads)
        const long long n = ((long long)sets.q_off[sets.n] - sets.q_off[0]) * a.q.heads;
        if (p.binned && !(launch_fits(sets.units, 64) && launch_fits((long long)sets.n * a.k.heads * kBinShares, 1024) && launch_fits(n, head_dim / 4)))
            return kNoWork;
        if (!p.binned && !launch_fits(xcd_grid(sets.units * p.parts), 256)) return kNoWork;
        return p.part_bytes + p.list_bytes + p.tile_bytes;
    }
    const DensePlan p = dense_plan(dtype, head_dim, a, sets);
    if (!launch_fits(xcd_grid(sets.units * p.parts), 256)) return kNoWork;
    return p.parts == 1 ? 0 : parts_bytes(((long long)sets.q_off[sets.n] - sets.q_off[0]) * a.q.heads * p.parts, head_dim);
}
hipError_t launch_attention(int dtype, int head_dim, const AttentionLaunch& a, AttnSets& sets, hipStream_t s) {
    return dtype == PPG_F32    ? run_dim<float>(a, sets, dtype, head_dim, s)
           : dtype == PPG_BF16 ? run_dim<__bf16>(a, sets, dtype, head_dim, s)
                               : run_dim<_Float16>(a, sets, dtype, head_dim, s);
}

}  // namespace ppg
