// What stands around the attention between descriptor sets (attn_mfma.hip): rotary positions, block means, block selection.
// Sums are held in 32 bits or more; what is stored in fewer bits is rounded once, to nearest even.
#include "attn_tile.h"
#include "wave_util.h"

#include <algorithm>

namespace ppg {

// ---- element types ----
template <class T> __device__ __forceinline__ float to_float(T v) { return (float)v; }
template <class T> struct alignas(16) Vec16 { T v[16 / sizeof(T)]; };

// cos and sin of `turns` full turns: the reduction is exact in 64 bits (the distance to the nearest quarter turn), the rest,
// at most an eighth of a turn, goes through the Taylor sums of sine and cosine, whose first terms left out are below 2^-29
__device__ __forceinline__ void cos_sin_turns(double turns, float& c, float& s) {
    const double quarter = rint(turns * 4.0);
    const float x = (float)((turns - quarter * 0.25) * 6.283185307179586476925);
    const float z = x * x;
    const float sn = x * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), 1.f);
    const float cs = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
    const int q = (int)(quarter - 4.0 * floor(quarter * 0.25));
    const float a = (q & 1) ? sn : cs, b = (q & 1) ? cs : sn;
    c = (q == 1 || q == 2) ? -a : a;
    s = (q >= 2) ? -b : b;
}

// ---- rotary positions ----
// Bound by memory: 64 streams of 1024 + 1024 rows, 4 heads of 64, bf16: 115 MB in 25 us, 4.6 TB/s (a copy reaches 5.1).
// A work-group turns RB rows of one tensor: the cosines and sines of its (row, pair)s go to LDS once and serve every head,
// then a thread takes 16 bytes at a time.
//   kInterleaved  a chunk holds whole pairs
//   kHalves       half of the turned part is whole chunks: a thread takes a chunk and the one its partners are in
//   kStaged       it is not (rot_dim = head_dim - 4, say): the rows pass through LDS, from where a chunk's partners are picked
enum RotaryForm { kInterleaved, kHalves, kStaged };
template <class T, int D, int RB, int FORM>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryLaunch a, int tiles0) {
    constexpr int N = 16 / (int)sizeof(T), CPR = D / N, PITCH = D + 2;
    extern __shared__ char lds[];
    float2* turn = (float2*)lds;                      // [RB][rot_dim / 2]
    const int half = a.rot_dim / 2, t = (int)blockIdx.x >= tiles0, row0 = ((int)blockIdx.x - (t ? tiles0 : 0)) * RB;
    T* stage = (T*)(lds + RB * (size_t)half * sizeof(float2));   // kStaged: [RB * heads of a round][PITCH]
    const int rows = min(RB, a.n_rows[t] - row0), heads = a.src[t].heads;
    const T* src = (const T*)a.src[t].p + (long long)row0 * a.src[t].row;
    T* dst = (T*)a.dst[t].p + (long long)row0 * a.dst[t].row;
    for (int i = threadIdx.x; i < rows * half; i += 256) {
        const int r = i / half, j = i % half;
        const float pos = a.pos[t][(long long)(row0 + r) * a.n_axes + (a.n_axes == 2 && j >= half / 2)];
        float2 cs;
        cos_sin_turns((double)pos * a.freq[j] * 0.15915494309189533577, cs.x, cs.y);
        if (a.inverse) cs.y = -cs.y;
        turn[i] = cs;
    }
    __syncthreads();
    if constexpr (FORM == kStaged) {
        // rounds of as many (row, head) vectors as the stage holds; a chunk is written only after all of its round was read
        constexpr int VR = 256 / CPR;
        for (int v0 = 0; v0 < rows * heads; v0 += VR) {
            const int v = v0 + threadIdx.x / CPR, ch = threadIdx.x % CPR;
            const bool on = v < rows * heads;
            const int r = on ? v / heads : 0, h = on ? v % heads : 0;
            Vec16<T> x;
            T* mine = stage + (threadIdx.x / CPR) * PITCH;
            if (on) {
                x = *(const Vec16<T>*)(src + r * a.src[t].row + h * a.src[t].head + ch * N);
#pragma unroll
                for (int e = 0; e < N; e++) mine[ch * N + e] = x.v[e];
            }
            __syncthreads();
            if (on) {
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const int d = ch * N + e;
                    if (d < a.rot_dim) {
                        const bool low = d < half;
                        const float2 cs = turn[r * half + (low ? d : d - half)];
                        const float u = to_float(x.v[e]), w = to_float(mine[low ? d + half : d - half]);
                        x.v[e] = (T)(low ? u * cs.x - w * cs.y : w * cs.y + u * cs.x);
                    }
                }
                *(Vec16<T>*)(dst + r * a.dst[t].row + h * a.dst[t].head + ch * N) = x;
            }
            __syncthreads();
        }
    } else {
        const int cut = a.rot_dim / N;   // kHalves: whole chunks turned; those behind are copied
        const int units = FORM == kHalves ? cut / 2 + (CPR - cut) : CPR;
        for (int i = threadIdx.x; i < rows * heads * units; i += 256) {
            const int u = i % units, v = i / units, h = v % heads, r = v / heads;
            const T* x = src + r * a.src[t].row + h * a.src[t].head;
            T* y = dst + r * a.dst[t].row + h * a.dst[t].head;
            if constexpr (FORM == kHalves) {
                if (u >= cut / 2) {
                    const int ch = u + cut / 2;
                    *(Vec16<T>*)(y + ch * N) = *(const Vec16<T>*)(x + ch * N);
                    continue;
                }
                Vec16<T> p = *(const Vec16<T>*)(x + u * N), q = *(const Vec16<T>*)(x + half + u * N);
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const float2 cs = turn[r * half + u * N + e];
                    const float f = to_float(p.v[e]), g = to_float(q.v[e]);
                    p.v[e] = (T)(f * cs.x - g * cs.y);
                    q.v[e] = (T)(f * cs.y + g * cs.x);
                }
                *(Vec16<T>*)(y + u * N) = p;
                *(Vec16<T>*)(y + half + u * N) = q;
            } else {
                Vec16<T> p = *(const Vec16<T>*)(x + u * N);
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const int j = (u * N + e) / 2;
                    if (j < half) {
                        const float2 cs = turn[r * half + j];
                        const float f = to_float(p.v[e]), g = to_float(p.v[e + 1]);
                        p.v[e] = (T)(f * cs.x - g * cs.y);
                        p.v[e + 1] = (T)(f * cs.y + g * cs.x);
                    }
                }
                *(Vec16<T>*)(y + u * N) = p;
            }
        }
    }
}

// ---- block means ----
// Bound by memory: 1000003 keys, 4 heads of 64, bf16: 529 MB in 93 us, 5.7 TB/s.
// One work-group per block.  The block's rows are taken 16 bytes at a time: a thread owns one chunk position and every
// `lanes`-th row, sums in 64 bits (the sum of 128 numbers of 8 or 11 bits is exact while their exponents span less than 35 steps),
// and the partial sums of a position meet in LDS.
template <class T, int D, class Sets>
__global__ __launch_bounds__(256) void block_means_kernel(BlockMeansLaunch a, Sets sets) {
    constexpr int N = 16 / (int)sizeof(T), CPR = D / N;
    __shared__ double part[256][N];
    __shared__ unsigned char keep[128];
    __shared__ int kept[2];
    const int b = blockIdx.x, tid = threadIdx.x;
    const SetHere set = set_of_block(sets, b, tid & 63);
    const int at = (b - set.blk0) * a.block, first = set.k0 + at, n = min(a.block, set.nk - at);
    if (tid < 128) {
        const bool on = tid < n && !(a.skip && a.skip[first + tid]);
        keep[tid] = on;
        const unsigned long long m = __ballot(on);
        if ((tid & 63) == 0) kept[tid >> 6] = __popcll(m);
    }
    __syncthreads();
    const int count = kept[0] + kept[1];
    if (tid == 0) a.count[b] = count;
    const int chunks = a.k.heads * CPR;
    for (int c0 = 0; c0 < chunks; c0 += 256) {
        const int width = min(256, chunks - c0), lanes = 256 / width;   // positions of this round, rows at a time
        const int c = tid % width, r0 = tid / width, h = (c0 + c) / CPR;
        double sum[N] = {};
        if (r0 < lanes) {
            const T* x = (const T*)a.k.p + (long long)first * a.k.row + h * a.k.head + (c0 + c) % CPR * N;
            // four rows in flight; what a skipped row holds, NaN included, counts as zero
            for (int r = r0; r < n; r += 4 * lanes) {
                Vec16<T> v[4];
                bool on[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int rr = r + i * lanes;
                    v[i] = *(const Vec16<T>*)(x + (long long)min(rr, n - 1) * a.k.row);
                    on[i] = rr < n && keep[rr];
                }
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < N; e++) sum[e] += on[i] ? (double)to_float(v[i].v[e]) : 0.0;
            }
        }
#pragma unroll
        for (int e = 0; e < N; e++) part[tid][e] = sum[e];
        __syncthreads();
        for (int i = tid; i < width * N; i += 256) {
            const int p = i / N, e = i % N;
            double total = 0;
            for (int l = 0; l < lanes; l++) total += part[l * width + p][e];
            a.mean[(long long)b * a.k.heads * D + (long long)c0 * N + i] = count ? (float)(total / count) : 0.f;
        }
        __syncthreads();
    }
}

// ---- block selection ----
// Scores become whole numbers in their order, so that (score, block) pairs compare exactly: larger first, the lower block
// first among equals.  0 marks a block that cannot be selected, NaN ranks as 1.
__device__ __forceinline__ unsigned long long score_key(double s) {
    if (s != s) return 1;
    const unsigned long long b = __double_as_longlong(s + 0.0);   // -0 is 0
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
struct Scored {
    unsigned long long key;
    int idx;
};
__device__ __forceinline__ bool scored_before(const Scored& a, const Scored& b) { return a.key > b.key || (a.key == b.key && a.idx < b.idx); }
// what lane l (the same for all) holds, without a trip through LDS
__device__ __forceinline__ double lane_value(double x, int l) {
    const long long b = __double_as_longlong(x);
    const unsigned lo = __builtin_amdgcn_readlane((int)b, l), hi = __builtin_amdgcn_readlane((int)(b >> 32), l);
    return __longlong_as_double((long long)(((unsigned long long)hi << 32) | lo));
}
__device__ __forceinline__ float lane_value(float x, int l) { return __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(x), l)); }
__device__ __forceinline__ Scored scored_lane(const Scored& a, int l) {
    const unsigned lo = __builtin_amdgcn_readlane((int)a.key, l), hi = __builtin_amdgcn_readlane((int)(a.key >> 32), l);
    return Scored{((unsigned long long)hi << 32) | lo, __builtin_amdgcn_readlane(a.idx, l)};
}
__device__ __forceinline__ Scored scored_shfl(const Scored& a, int lane) {
    Scored r;
    r.key = __shfl(a.key, lane);
    r.idx = __shfl(a.idx, lane);
    return r;
}
// one compare-exchange step of a bitonic network over the 64 lanes; up: this lane keeps the earlier of the two
__device__ __forceinline__ void scored_step(Scored& a, int lane, int dist, bool up) {
    const Scored o = scored_shfl(a, lane ^ dist);
    const bool lower = !(lane & dist);
    if (scored_before(o, a) == (lower == up)) a = o;
}
__device__ __forceinline__ void scored_sort(Scored& a, int lane) {
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) scored_step(a, lane, j, !(lane & k));
}

// The plain way, a wave per (query row, key head): a lane scores one block in 64 bits; the best n_sel so far are kept one per
// lane, in order, and 64 new ones are merged in only when one of them beats the last of those.  q: the summed query, component
// d in lane d % 64, place d / 64.
template <int D>
__device__ Scored select_all(const double (&q)[(D + 63) / 64][1], const float* mean, const int* count, int nb, int kv_heads, int n_sel, int lane) {
    Scored best{0, 0x7fffffff};
    for (int b0 = 0; b0 < nb; b0 += 64) {
        const int b = b0 + lane;
        const bool on = b < nb && count[b] > 0;
        const float* m = mean + (long long)(on ? b : 0) * kv_heads * D;
        double dot = 0;
        for (int d = 0; d < D; d++) dot = fma(lane_value(q[d >> 6][0], d & 63), (double)m[d], dot);
        const Scored c = on ? Scored{score_key(dot), b} : Scored{0, 0x7fffffff};
        const Scored worst = scored_lane(best, n_sel - 1);
        if (!__any(scored_before(c, worst))) continue;
        Scored x = c;
        scored_sort(x, lane);
        // the 64 best of two ordered lists: the better of every mirrored pair, which leaves a bitonic row
        const Scored o = scored_shfl(x, 63 - lane);
        if (scored_before(o, best)) best = o;
#pragma unroll
        for (int j = 32; j > 0; j >>= 1) scored_step(best, lane, j, true);
    }
    return best;
}

// float as a whole number in its order, and back; what no finite number gives becomes the nearest of them
__device__ __forceinline__ unsigned float_key(float f) {
    const unsigned b = __float_as_uint(f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_float(unsigned k) {
    k = max(0x00800000u, min(k, 0xff7fffffu));
    return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}

// A work-group selects for ROWS query rows of one (set, key head).  The products of all of them with a stretch of blocks come from the
// bf16 matrix unit, both inputs split into two halves and three of the four products taken: off by at most
// E = 2^-13 |q| |mean| (Cauchy-Schwarz; what is left out is below 3 * 2^-16, the 32-bit sums of up to 384 terms below
// 2^-15).  They stay in LDS.  Then a wave takes a row: the n_sel-th largest of (product - E) is a bound t that the n_sel best
// blocks reach for sure, so only blocks with product + E >= t can be among them.  Mostly those are n_sel and that is the
// answer; else they are scored in 64 bits and ranked exactly.  Rows for which that does not hold together (a product that is
// not finite, more than 128 left, as with many equal means, or a vector shorter than 1e-12 that is not zero) go the plain way.
// 8 streams of 1024 rows against 65537 keys (1025 blocks), 4 heads of 64: 104 us, of which the products take half (the conversion of
// the means to bf16 halves, repeated for every 32 rows, and the latency of the L2) and the choice the other half (some 600
// vector instructions a row); all products in 64 bits on their matrix unit would be 61 us without any choice.  128 components,
// 960 blocks: 232 us.  1024 threads leave a wave 128 registers, and every form spills: 15 vector registers at 64 components and 1088 blocks, 64 at
// 128 (there in the loop over the rows), and scalar ones, most of them in the plain way's loop.
constexpr int kSelWaves = 16;
// A vector that is not zero has at least this for its squares' sum (they vanish in 32 bits below 2^-75): far below where the bound is
// given up (1e-24), far above zero.
constexpr float kNoSquare = 1e-30f;
// A row's scores, and once its wave has them in registers, that wave's notes: the blocks left, their bounds, their exact keys.
template <int PER> union SelectRow {
    float score[PER * 64 + 4];
    struct {
        unsigned short cand[128];
        float low[128], high[128];
        unsigned long long key[128];
        unsigned long long best_key[64];
        int best_idx[64];
    } note;
};
template <int D, int ROWS, int PER> struct SelectLds {
    SelectRow<PER> row[ROWS];
    float norm[PER * 64];                 // |mean|, -1 for a block that cannot be selected
    char q[2][ROWS * D * 2];           // the summed queries' upper and lower halves, chunks permuted against bank conflicts
};
template <class T, int D, int ROWS, int PER, class Sets>
__global__ __launch_bounds__(1024, 4) void block_select_kernel(BlockSelectLaunch a, Sets sets) {
    constexpr int CHUNK = PER * 64, RPW = ROWS / kSelWaves, N = 16 / (int)sizeof(T);
    constexpr int LPC = D / 16, CPP = 64 / LPC;   // lanes that share a candidate's product, candidates of a pass
    __shared__ alignas(16) SelectLds<D, ROWS, PER> lds;
    const Launch here = launch_of(sets);
    const int unit = xcd_unit(blockIdx.x, here.units);
    if (unit >= here.units) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const SetHere set = set_of_tile(sets, unit, lane);
    const int q0 = set.q0, nq = set.nq;
    // the heads in turn: work-groups that run at the same time then read whole rows of means between them, and with those all
    // channels of the L2
    const int g = (unit - set.tile0) % a.kv_heads, row0 = ((unit - set.tile0) / a.kv_heads) * ROWS;
    const int group = a.q.heads / a.kv_heads, nb = set.blocks;
    const float* mean = a.mean + ((long long)set.blk0 * a.kv_heads + g) * D;
    const long long stride = (long long)a.kv_heads * D;
    const int* count = a.count + set.blk0;
    auto query = [&](int row, int h) { return (const T*)a.q.p + (long long)(q0 + min(row, nq - 1)) * a.q.row + ((long long)g * group + h) * a.q.head; };
    auto q_chunk = [&](int half, int r, int ch) { return lds.q[half] + r * (D * 2) + ((ch ^ (r & (D >= 64 ? 7 : 3))) << 4); };

    f32x4 mx[D / 32][2];
    bool alive = false;
    auto load = [&](int b0, int t) {
        const int n = min(CHUNK, nb - b0), b = t * 16 + (lane & 15), bb = b0 + min(b, n - 1);
        const float* m = mean + bb * stride + (lane >> 4) * 8;
#pragma unroll
        for (int k = 0; k < D / 32; k++) {
            mx[k][0] = *(const f32x4*)(m + k * 32);
            mx[k][1] = *(const f32x4*)(m + k * 32 + 4);
        }
        alive = b < n && count[bb] > 0;
    };
    if (wave * 16 < nb) load(0, wave);   // (in flight while the queries are prepared)

    // a wave per RPW rows: the group's sum, its halves to LDS, its length
    Scored best[RPW];
    float eq[RPW];   // 2^-13 |q|, NaN: the plain way
#pragma unroll
    for (int i = 0; i < RPW; i++) {
        const int r = wave * RPW + i;
        float sq = 0.f;
        for (int d = lane; d < D; d += 64) {
            double x = 0;
            for (int h = 0; h < group; h++) x += (double)to_float(query(row0 + r, h)[d]);
            const __bf16 hi = (__bf16)(float)x, lo = (__bf16)(float)(x - (double)(float)hi);
            *(__bf16*)(q_chunk(0, r, d >> 3) + (d & 7) * 2) = hi;
            *(__bf16*)(q_chunk(1, r, d >> 3) + (d & 7) * 2) = lo;
            sq = fmaf((float)x, (float)x, sq);
            if (x != 0 && sq < kNoSquare) sq = kNoSquare;
        }
        sq = wave_sum(sq);
        // (one so short that its components leave bf16's range has no such bound, unless it is zero)
        eq[i] = sq < 1e36f && !(sq < 1e-24f && sq > 0.f) ? sqrtf(sq) * 1.2208e-4f : NAN;
        best[i] = Scored{0, 0x7fffffff};
    }

    for (int b0 = 0; b0 < nb; b0 += CHUNK) {
        const int n = min(CHUNK, nb - b0);
        if (b0 && wave * 16 < n) load(b0, wave);
        __syncthreads();   // the queries are in LDS; the last stretch has been read
        for (int t = wave; t * 16 < n; t += kSelWaves) {
            f32x4 acc[RPW] = {};
            float sm = 0.f;
            bf16x8 mh[D / 32], ml[D / 32];
#pragma unroll
            for (int k = 0; k < D / 32; k++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float x = mx[k][e / 4][e % 4];
                    mh[k][e] = (__bf16)x;
                    ml[k][e] = (__bf16)(x - (float)mh[k][e]);
                    sm = fmaf(x, x, sm);
                }
            if (__any(sm < kNoSquare)) {   // hardly ever: the mean of a block without keys
                bool any = false;
#pragma unroll
                for (int k = 0; k < D / 32; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) any |= mx[k][e / 4][e % 4] != 0.f;
                if (any && sm < kNoSquare) sm = kNoSquare;
            }
            const bool on = alive;
            if ((t + kSelWaves) * 16 < n) load(b0, t + kSelWaves);
#pragma unroll
            for (int rt = 0; rt < RPW; rt++) {
#pragma unroll
                for (int k = 0; k < D / 32; k++) {
                    const int r = rt * 16 + (lane & 15), ch = k * 4 + (lane >> 4);
                    const bf16x8 qh = *(const bf16x8*)q_chunk(0, r, ch), ql = *(const bf16x8*)q_chunk(1, r, ch);
                    acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mh[k], qh, acc[rt], 0, 0, 0);
                    acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mh[k], ql, acc[rt], 0, 0, 0);
                    acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ml[k], qh, acc[rt], 0, 0, 0);
                }
                *(f32x4*)&lds.row[rt * 16 + (lane & 15)].score[t * 16 + (lane >> 4) * 4] = acc[rt];
            }
            sm += __shfl_xor(sm, 16);
            sm += __shfl_xor(sm, 32);
            // (as short a mean as the query above: NaN, which sends the rows the plain way)
            if (lane < 16) lds.norm[t * 16 + lane] = on ? (sm < 1e-24f && sm > 0.f ? NAN : sqrtf(sm) * 1.0001f) : -1.f;
        }
        for (int b = (n + 15) / 16 * 16 + threadIdx.x; b < CHUNK; b += 1024) lds.norm[b] = -1.f;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RPW; i++) {
            const int row = wave * RPW + i;
            if (eq[i] != eq[i] || row0 + row >= nq) continue;   // the same for all lanes
            float low[PER], high[PER], top = -INFINITY;
            bool odd = false;
#pragma unroll
            for (int p = 0; p < PER; p++) {
                const float x = lds.row[row].score[p * 64 + lane], nm = lds.norm[p * 64 + lane], e = nm * eq[i];
                const bool on = !(nm < 0.f);
                odd |= on && !(fabsf(x) + e < 3e38f);
                low[p] = on ? x - e : -INFINITY;
                high[p] = on ? x + e : -INFINITY;
                top = fmaxf(top, low[p]);
            }
            if (__any(odd)) {
                eq[i] = NAN;
                continue;
            }
            // a bound that n_sel blocks reach: the n_sel-th largest of the lanes' largest, to 18 of its 32 bits (or, with fewer
            // blocks, the lowest number)
            const unsigned top_key = top == -INFINITY ? 0 : float_key(top);
            unsigned tk = 0;
            for (int bit = 31; bit >= 14; bit--) {
                const unsigned c = tk | (1u << bit);
                if (__popcll(__ballot(top_key >= c)) >= a.n_sel) tk = c;
            }
            float t = key_float(tk);
            auto passing = [&](const float (&x)[PER], float from) {
                int c = 0;
#pragma unroll
                for (int p = 0; p < PER; p++) c += __popcll(__ballot(x[p] >= from));
                return c;
            };
            int left = passing(high, t);
            if (left > 128) {   // long lists: the n_sel-th largest of all
                tk = 0;
                for (int bit = 31; bit >= 0; bit--) {
                    const unsigned c = tk | (1u << bit);
                    if (passing(low, key_float(c)) >= a.n_sel) tk = c;
                }
                t = key_float(tk);
                left = passing(high, t);
            }
            if (left > 128) {
                eq[i] = NAN;
                continue;
            }
            // (LDS serves a wave in order, and nobody else touches this row any more)
            auto& note = lds.row[row].note;
            __builtin_amdgcn_wave_barrier();
            int at = 0;
#pragma unroll
            for (int p = 0; p < PER; p++) {
                const bool on = high[p] >= t;
                const unsigned long long m = __ballot(on);
                if (on) {
                    const int to = at + bits_below(m);
                    note.cand[to] = (unsigned short)(p * 64 + lane);
                    note.low[to] = low[p];
                    note.high[to] = high[p];
                }
                at += __popcll(m);
            }
            __builtin_amdgcn_wave_barrier();
            int cand[2];
            unsigned long long key[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                cand[k] = k * 64 + lane < left ? note.cand[k * 64 + lane] : -1;
                key[k] = 1;
            }
            bool in[2] = {cand[0] >= 0, cand[1] >= 0};
            if (left > a.n_sel) {
                // the bound once more, exactly: the largest that n_sel of what is left reach
                float lo[2], hi[2];
                int reach[2] = {0, 0};
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    lo[k] = in[k] ? note.low[k * 64 + lane] : -INFINITY;
                    hi[k] = in[k] ? note.high[k * 64 + lane] : -INFINITY;
                }
                if (left <= 64) {
                    for (int l = 0; l < left; l++) reach[0] += lane_value(lo[0], l) >= lo[0];
                } else {
#pragma unroll
                    for (int k = 0; k < 2; k++)
                        for (int l = 0; l < min(left - 64 * k, 64); l++) {
                            const float o = lane_value(lo[k], l);
                            reach[0] += o >= lo[0];
                            reach[1] += o >= lo[1];
                        }
                }
                t = wave_max(fmaxf(in[0] && reach[0] >= a.n_sel ? lo[0] : -INFINITY, in[1] && reach[1] >= a.n_sel ? lo[1] : -INFINITY));
                int kept = 0;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    in[k] = in[k] && hi[k] >= t;
                    const unsigned long long m = __ballot(in[k]);
                    if (in[k]) note.cand[kept + bits_below(m)] = (unsigned short)cand[k];
                    kept += __popcll(m);
                }
                __builtin_amdgcn_wave_barrier();
                left = kept;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    in[k] = k * 64 + lane < left;
                    cand[k] = in[k] ? note.cand[k * 64 + lane] : -1;
                }
            }
            const bool choose = b0 || nb > CHUNK || left > a.n_sel;   // (keys for the stretches to come, too)
            if (!choose) {
                best[i] = in[0] ? Scored{1, cand[0]} : Scored{0, 0x7fffffff};   // (at most n_sel of them, in order)
                continue;
            }
            int order[3] = {0, 0, 0};
            {
                double q[16];
#pragma unroll
                for (int e = 0; e < 16; e++) q[e] = 0;
                for (int h = 0; h < group; h++)
#pragma unroll
                    for (int v = 0; v < 16 / N; v++) {
                        const Vec16<T> y = *(const Vec16<T>*)(query(row0 + row, h) + (lane % LPC) * 16 + v * N);
#pragma unroll
                        for (int e = 0; e < N; e++) q[v * N + e] += (double)to_float(y.v[e]);
                    }
                for (int c0 = 0; c0 < left; c0 += CPP) {
                    const int c = c0 + lane / LPC, b = b0 + note.cand[min(c, left - 1)];
                    const float* m = mean + b * stride + (lane % LPC) * 16;
                    f32x4 x[4];
#pragma unroll
                    for (int v = 0; v < 4; v++) x[v] = *(const f32x4*)(m + 4 * v);
                    double dot = 0;
#pragma unroll
                    for (int e = 0; e < 16; e++) dot = fma(q[e], (double)x[e / 4][e % 4], dot);
#pragma unroll
                    for (int w = 1; w < LPC; w <<= 1) dot += __shfl_xor(dot, w);
                    if (lane % LPC == 0 && c < left) note.key[c] = score_key(dot);
                }
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int k = 0; k < 2; k++)
                    if (in[k]) key[k] = note.key[k * 64 + lane];
            }
            // ranks among these and the best of the stretches before; every list is in ascending block order already
            const Scored all[3] = {best[i], in[0] ? Scored{key[0], b0 + cand[0]} : Scored{0, 0x7fffffff},
                                   in[1] ? Scored{key[1], b0 + cand[1]} : Scored{0, 0x7fffffff}};
            {
                const int sizes[3] = {b0 ? a.n_sel : 0, min(left, 64), left - 64};
#pragma unroll
                for (int k = 0; k < 3; k++)
                    for (int l = 0; l < sizes[k]; l++) {
                        const Scored o = scored_lane(all[k], l);
#pragma unroll
                        for (int x = 0; x < 3; x++) order[x] += scored_before(o, all[x]);
                    }
            }
            // the n_sel first, by block: the earlier stretches', then these
            int to = 0;
#pragma unroll
            for (int k = 0; k < 3; k++) {
                const bool take = all[k].idx != 0x7fffffff && order[k] < a.n_sel;
                const unsigned long long m = __ballot(take);
                const int place = to + bits_below(m);
                if (take) {
                    note.best_key[place] = all[k].key;
                    note.best_idx[place] = all[k].idx;
                }
                to += __popcll(m);
            }
            __builtin_amdgcn_wave_barrier();
            best[i] = lane < to ? Scored{note.best_key[lane], note.best_idx[lane]} : Scored{0, 0x7fffffff};
            __builtin_amdgcn_wave_barrier();
        }
    }
#pragma unroll
    for (int i = 0; i < RPW; i++) {
        const int row = row0 + wave * RPW + i;
        if (row >= nq) continue;
        if (eq[i] != eq[i]) {
            double q[(D + 63) / 64][1];
#pragma unroll
            for (int k = 0; k < (D + 63) / 64; k++) {
                q[k][0] = 0;
                for (int h = 0; h < group; h++) q[k][0] += (double)to_float(query(row, h)[min(k * 64 + lane, D - 1)]);
            }
            Scored x{0, 0x7fffffff};
            const Scored b = select_all<D>(q, mean, count, nb, a.kv_heads, a.n_sel, lane);
            if (lane < a.n_sel) x.idx = b.idx;
            scored_sort(x, lane);
            best[i] = x;
        }
        if (lane < a.n_sel) a.sel[((long long)(q0 + row) * a.kv_heads + g) * a.n_sel + lane] = best[i].idx == 0x7fffffff ? -1 : best[i].idx;
    }
}

// ---- launches ----
#define BY_TYPE(dtype, CALL)                                    \
    do {                                                        \
        if (dtype == PPG_F32) { using T = float; CALL; }        \
        else if (dtype == PPG_BF16) { using T = __bf16; CALL; } \
        else { using T = _Float16; CALL; }                      \
    } while (0)
#define BY_DIM(dim, CALL)                                     \
    do {                                                      \
        if (dim == 32) { constexpr int D = 32; CALL; }        \
        else if (dim == 64) { constexpr int D = 64; CALL; }   \
        else { constexpr int D = 128; CALL; }                 \
    } while (0)

bool rotary_fits(const RotaryLaunch& a) { return launch_fits(((long long)a.n_rows[0] + 15) / 16 + ((long long)a.n_rows[1] + 15) / 16, 256); }
hipError_t launch_rotary(int dtype, const RotaryLaunch& a, hipStream_t s) {
    const long long rows = (long long)a.n_rows[0] + a.n_rows[1];
    if (!rows) return hipSuccess;
    const int n = dtype == PPG_F32 ? 4 : 8, half = a.rot_dim / 2;
    const int form = a.layout == PPG_ROTARY_INTERLEAVED ? kInterleaved : half % n == 0 ? kHalves : kStaged;
    auto go = [&](auto kernel, int rb, size_t stage) {
        const int t0 = (int)(((long long)a.n_rows[0] + rb - 1) / rb), t1 = (int)(((long long)a.n_rows[1] + rb - 1) / rb);
        kernel<<<(unsigned)t0 + (unsigned)t1, 256, rb * (size_t)half * sizeof(float2) + stage, s>>>(a, t0);
        return hipGetLastError();
    };
    hipError_t e = hipSuccess;
    // few rows: four to a work-group, so that more of them run; many: sixteen, so that a work-group has enough to load
#define FORMS(RB)                                                                                                              \
    BY_TYPE(dtype, BY_DIM(a.head_dim, (e = form == kInterleaved ? go(rotary_kernel<T, D, RB, kInterleaved>, RB, 0)             \
                                           : form == kHalves    ? go(rotary_kernel<T, D, RB, kHalves>, RB, 0)                  \
                                                                : go(rotary_kernel<T, D, RB, kStaged>, RB,                     \
                                                                     (size_t)256 / (D * sizeof(T) / 16) * (D + 2) * sizeof(T)))))
    if (rows < 16384) FORMS(4);
    else FORMS(16);
#undef FORMS
    return e;
}

bool block_means_fits(const AttnSets& sets) { return launch_fits(sets.blk[sets.n], 256); }
hipError_t launch_block_means(int dtype, int head_dim, const BlockMeansLaunch& a, AttnSets& sets, hipStream_t s) {
    const int nb = sets.blk[sets.n];
    if (!nb) return hipSuccess;
    return with_sets(sets, [&](const auto& st) {
        using Sets = std::decay_t<decltype(st)>;
        BY_TYPE(dtype, BY_DIM(head_dim, (block_means_kernel<T, D, Sets><<<nb, 256, 0, s>>>(a, st))));
        return hipGetLastError();
    });
}

static int select_tiles(const BlockSelectLaunch& a, AttnSets& sets, int rows) {
    sets.tile[0] = 0;
    for (int i = 0; i < sets.n; i++)
        sets.tile[i + 1] = sets.tile[i] + (int)(((long long)sets.q_off[i + 1] - sets.q_off[i] + rows - 1) / rows * a.kv_heads);
    return end_tiles(sets);
}
bool block_select_fits(const BlockSelectLaunch& a, AttnSets& sets) { return launch_fits(xcd_grid(select_tiles(a, sets, 32)), 1024); }
hipError_t launch_block_select(int dtype, int head_dim, const BlockSelectLaunch& a, AttnSets& sets, hipStream_t s) {
    int most = 0;
    for (int i = 0; i < sets.n; i++) most = std::max(most, sets.blk[i + 1] - sets.blk[i]);
    // a row per wave where that still leaves CUs without work (one frame of 500 rows, 4 heads, 313 blocks: 13 us, 23 us with two), else two, which read
    // the means half as often (8 streams of 1024 rows: 104 us, 149 us with one); few blocks: as many registers as those take, up to
    // 320 (8 streams of 1024 rows, 4 heads of 64 bf16, with room for 320 : for 1088: 172 blocks 62 : 73 us, 320 blocks 69 : 79; beyond, in
    // several stretches, 321 blocks 136 : 80, 640 blocks 173 : 93; one frame 320 blocks 13.1 : 15.2, 321 blocks 20.6 : 15.1)
#define SELECT(ROWS, PER)                                                                                                                      \
    return with_sets(sets, [&](const auto& st) {                                                                                               \
        BY_TYPE(dtype, BY_DIM(head_dim, (block_select_kernel<T, D, ROWS, PER, std::decay_t<decltype(st)>><<<xcd_grid(sets.units), 1024, 0, s>>>(a, st)))); \
        return hipGetLastError();                                                                                                              \
    })
    if (select_tiles(a, sets, 32) >= 256) {
        if (most <= 5 * 64) SELECT(32, 5);
        else SELECT(32, 17);
    } else if (!select_tiles(a, sets, 16)) return hipSuccess;
    else if (most <= 5 * 64) SELECT(16, 5);
    else SELECT(16, 17);
#undef SELECT
}

}  // namespace ppg
