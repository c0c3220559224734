// What stands around the attention between descriptor sets (attn_mfma.hip): rotary positions, block means, block selection.
// Sums are held in 32 bits or more; what is stored in fewer bits is rounded once, to nearest even.
#include "attn_tile.h"
#include "wave_util.h"

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
// One thread per pair, and per component that is only copied.
template <class T>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryLaunch a, long long units0, long long units1) {
    const int half = a.rot_dim / 2, rest = a.head_dim - a.rot_dim, per_head = half + rest;
    long long u = (long long)blockIdx.x * 256 + threadIdx.x;
    const int t = u >= units0;
    if (t) u -= units0;
    if (u >= (t ? units1 : units0)) return;
    const int j = (int)(u % per_head);
    const long long rh = u / per_head;
    const int h = (int)(rh % a.src[t].heads);
    const long long r = rh / a.src[t].heads;
    const T* x = (const T*)a.src[t].p + r * a.src[t].row + h * a.src[t].head;
    T* y = (T*)a.dst[t].p + r * a.dst[t].row + h * a.dst[t].head;
    if (j >= half) {
        const int i = a.rot_dim + (j - half);
        y[i] = x[i];
        return;
    }
    const int axis = a.n_axes == 2 && j >= half / 2;
    float c, s;
    cos_sin_turns((double)a.pos[t][r * a.n_axes + axis] * a.freq[j] * 0.15915494309189533577, c, s);
    if (a.inverse) s = -s;
    const int i0 = a.layout == PPG_ROTARY_HALF ? j : 2 * j, i1 = a.layout == PPG_ROTARY_HALF ? j + half : 2 * j + 1;
    const float u0 = to_float(x[i0]), u1 = to_float(x[i1]);
    y[i0] = (T)(u0 * c - u1 * s);
    y[i1] = (T)(u0 * s + u1 * c);
}

// ---- block means ----
// One thread per (block, head, component).
template <class T>
__global__ __launch_bounds__(256) void block_means_kernel(BlockMeansLaunch a, AttnSets sets, int D) {
    const int b = blockIdx.x, s = find_set(sets.blk, sets.n, b);
    const int first = sets.k_off[s] + (b - sets.blk[s]) * a.block, last = min(first + a.block, sets.k_off[s + 1]);
    int n = last - first;
    if (a.skip) {
        n = 0;
        for (int r = first; r < last; r++) n += a.skip[r] == 0;
    }
    if (threadIdx.x == 0) a.count[b] = n;
    for (int i = threadIdx.x; i < a.k.heads * D; i += 256) {
        const T* x = (const T*)a.k.p + (i / D) * a.k.head + i % D;
        double sum = 0;
        for (int r = first; r < last; r++)
            if (!a.skip || a.skip[r] == 0) sum += (double)to_float(x[(long long)r * a.k.row]);
        a.mean[(long long)b * a.k.heads * D + i] = n ? (float)(sum / n) : 0.f;
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

// One wave per (query row, key head).  A lane scores one block; the best n_sel so far are kept one per lane, in order, and
// 64 new ones are merged in only when one of them beats the last of those.
template <class T>
__global__ __launch_bounds__(256) void block_select_kernel(BlockSelectLaunch a, AttnSets sets, int D) {
    __shared__ double qs[4][128];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long long unit = (long long)blockIdx.x * 4 + w;
    const long long rows = sets.q_off[sets.n] - sets.q_off[0];
    const bool live = unit < rows * a.kv_heads;
    const int r = sets.q_off[0] + (int)((live ? unit : 0) / a.kv_heads), g = (int)((live ? unit : 0) % a.kv_heads);
    const int group = a.q.heads / a.kv_heads;
    for (int d = lane; d < D; d += 64) {
        double sum = 0;
        for (int h = 0; h < group; h++) sum += (double)to_float(((const T*)a.q.p)[(long long)r * a.q.row + (g * group + h) * a.q.head + d]);
        qs[w][d] = sum;
    }
    __syncthreads();
    if (!live) return;
    const int s = find_set(sets.q_off, sets.n, r), nb = sets.blk[s + 1] - sets.blk[s];
    Scored best{0, 0x7fffffff};
    for (int b0 = 0; b0 < nb; b0 += 64) {
        const int b = b0 + lane;
        Scored c{0, 0x7fffffff};
        if (b < nb && a.count[sets.blk[s] + b] > 0) {
            const float* m = a.mean + ((long long)(sets.blk[s] + b) * a.kv_heads + g) * D;
            double dot = 0;
            for (int d = 0; d < D; d++) dot = fma(qs[w][d], (double)m[d], dot);
            c.key = score_key(dot);
            c.idx = b;
        }
        const Scored worst = scored_shfl(best, a.n_sel - 1);
        if (!__any(scored_before(c, worst))) continue;
        scored_sort(c, lane);
        // the 64 best of two ordered lists: the better of every mirrored pair, which leaves a bitonic row
        const Scored o = scored_shfl(c, 63 - lane);
        if (scored_before(o, best)) best = o;
#pragma unroll
        for (int j = 32; j > 0; j >>= 1) scored_step(best, lane, j, true);
    }
    // ascending by block
    Scored out{0, lane < a.n_sel ? best.idx : 0x7fffffff};
    scored_sort(out, lane);
    if (lane < a.n_sel) a.sel[((long long)r * a.kv_heads + g) * a.n_sel + lane] = out.idx == 0x7fffffff ? -1 : out.idx;
}

// ---- launches ----
#define BY_TYPE(dtype, CALL)                   \
    do {                                       \
        if (dtype == PPG_F32) { using T = float; CALL; }        \
        else if (dtype == PPG_BF16) { using T = __bf16; CALL; } \
        else { using T = _Float16; CALL; }     \
    } while (0)
hipError_t launch_rotary(int dtype, const RotaryLaunch& a, hipStream_t s) {
    const long long per_head = a.rot_dim / 2 + (a.head_dim - a.rot_dim);
    const long long u0 = a.n_rows[0] ? a.n_rows[0] * (long long)a.src[0].heads * per_head : 0;
    const long long u1 = a.n_rows[1] ? a.n_rows[1] * (long long)a.src[1].heads * per_head : 0;
    if (u0 + u1 == 0) return hipSuccess;
    const unsigned grid = (unsigned)((u0 + u1 + 255) / 256);
    BY_TYPE(dtype, (rotary_kernel<T><<<grid, 256, 0, s>>>(a, u0, u1)));
    return hipGetLastError();
}

hipError_t launch_block_means(int dtype, int head_dim, const BlockMeansLaunch& a, AttnSets& sets, hipStream_t s) {
    const int nb = sets.blk[sets.n];
    if (!nb) return hipSuccess;
    BY_TYPE(dtype, (block_means_kernel<T><<<nb, 256, 0, s>>>(a, sets, head_dim)));
    return hipGetLastError();
}

hipError_t launch_block_select(int dtype, int head_dim, const BlockSelectLaunch& a, AttnSets& sets, hipStream_t s) {
    const long long units = ((long long)sets.q_off[sets.n] - sets.q_off[0]) * a.kv_heads;
    if (!units) return hipSuccess;
    BY_TYPE(dtype, (block_select_kernel<T><<<(unsigned)((units + 3) / 4), 256, 0, s>>>(a, sets, head_dim)));
    return hipGetLastError();
}

}  // namespace ppg
