// Launch interface of the attention kernels (attn_kernels.hip) towards ppg_attn.cpp.  Everything was checked on the host
// before it gets here: types, sizes, strides, alignments, the offsets' order.
#pragma once
#include "../../include/ppgfront.h"
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ppg {

// HIP counts the threads of a launch in 32 bits
inline bool launch_fits(long long groups, int threads) { return groups * threads < (1LL << 32); }

// The sets of a call travel with the launch (kernel arguments): no copy to the device, nothing that a later call could
// overwrite, and a captured graph keeps its own.
// What a work-group reads of them comes one round trip to memory after the other, so these are kept few: the number of units
// stands in front, and the lists that are searched end in INT_MAX.
struct AttnSets {
    int n;
    int units = 0;   // tile[n]
    int q_off[PPG_ATTN_MAX_SETS + 1], k_off[PPG_ATTN_MAX_SETS + 1];
    int tile[PPG_ATTN_MAX_SETS + 1];   // first work-group tile of a set (what a tile is depends on the kernel)
    int blk[PPG_ATTN_MAX_SETS + 1];    // first key block of a set
};
// One set alone (or, where no kernel asks which set a row is in, all of them as one): 24 bytes of arguments instead of 2 KB, which
// take the host 1.3 us less to launch.
struct OneSet {
    int units, q0, q1, k0, k1, blocks;
    explicit OneSet(const AttnSets& s) : units(s.units), q0(s.q_off[0]), q1(s.q_off[s.n]), k0(s.k_off[0]), k1(s.k_off[s.n]), blocks(s.n == 1 ? s.blk[1] : 0) {}
};
template <class F> auto with_sets(const AttnSets& s, F f) { return s.n == 1 ? f(OneSet(s)) : f(s); }
// INT_MAX behind the last set
inline void end_list(const AttnSets& sets, int (&list)[PPG_ATTN_MAX_SETS + 1]) {
    if (sets.n > 1) for (int i = sets.n + 1; i <= PPG_ATTN_MAX_SETS; i++) list[i] = 0x7fffffff;
}
inline int end_tiles(AttnSets& sets) {
    end_list(sets, sets.tile);
    return sets.units = sets.tile[sets.n];
}

struct RotaryLaunch {
    int head_dim, rot_dim, layout, inverse, n_axes;
    int n_rows[2];
    const float* pos[2];
    const double* freq;
    ppg_rows src[2], dst[2];
};
bool rotary_fits(const RotaryLaunch& a);   // one launch holds it (likewise below)
hipError_t launch_rotary(int dtype, const RotaryLaunch& a, hipStream_t s);

struct BlockMeansLaunch {
    int block;
    ppg_rows k;
    const uint8_t* skip;
    float* mean;
    int32_t* count;
};
bool block_means_fits(const AttnSets& sets);
hipError_t launch_block_means(int dtype, int head_dim, const BlockMeansLaunch& a, AttnSets& sets, hipStream_t s);

struct BlockSelectLaunch {
    int block, kv_heads, n_sel;
    ppg_rows q;
    const float* mean;
    const int32_t* count;
    int32_t* sel;
};
bool block_select_fits(const BlockSelectLaunch& a, AttnSets& sets);
hipError_t launch_block_select(int dtype, int head_dim, const BlockSelectLaunch& a, AttnSets& sets, hipStream_t s);

struct AttentionLaunch {
    float scale;
    ppg_rows q, k, v, out;
    const uint8_t* skip;
    float* lse;
    int block, n_sel;
    const int32_t* sel;
    void* work;
};
constexpr size_t kNoWork = ~(size_t)0;   // "one launch does not hold it"
size_t attention_work(int dtype, int head_dim, const AttentionLaunch& a, AttnSets& sets);
hipError_t launch_attention(int dtype, int head_dim, const AttentionLaunch& a, AttnSets& sets, hipStream_t s);

}  // namespace ppg
