// Host side of the attention entry points: argument checks, streams, launches.  C ABI in include/ppgfront.h.
// The arguments are checked before the context, so that what is refused, and why (ppg_last_error(NULL)), can be asked for
// without a GPU.
#include "ppg_ctx.h"
#include "attn_kernels.h"

namespace {

// Makes the context's GPU current for the duration of a call and the caller's again behind it.
struct DeviceScope {
    int before = -1;
    hipError_t err;
    explicit DeviceScope(int dev) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != dev) err = hipSetDevice(dev);
        else before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

size_t elem_size(int dtype) { return dtype == PPG_F32 ? 4 : 2; }

// 0, or the reason why these rows cannot be used (output: strides must keep the vectors apart)
const char* rows_fault(const ppg_rows& r, int dtype, int head_dim, long long n_rows, bool output) {
    if (r.heads < 1 || r.heads > 65535) return "heads must be 1..65535";
    if (n_rows > 0 && !r.p) return "address is NULL";
    const long long e = (long long)elem_size(dtype);
    if ((uintptr_t)r.p % 16) return "address is not a multiple of 16";
    if (r.row < 0 || r.head < 0 || r.row > (1LL << 40) || r.head > (1LL << 40)) return "stride is negative or beyond 2^40";
    if (r.row * e % 16 || r.head * e % 16) return "a stride is not a multiple of 16 bytes";
    if (output && n_rows > 0) {
        const __int128 row = r.row, head = r.head;
        const bool rows_outer = (r.heads == 1 || head >= head_dim) && (n_rows == 1 || row >= (r.heads - 1) * head + head_dim);
        const bool heads_outer = (n_rows == 1 || row >= head_dim) && (r.heads == 1 || head >= (n_rows - 1) * row + head_dim);
        if (!rows_outer && !heads_outer) return "strides of an output make its vectors overlap";
    }
    return nullptr;
}

constexpr long long kMostVectors = (1LL << 31) - (1 << 10);   // rows times heads of a call: tiles that pass a set's end stay countable

bool known_type(int dtype) { return dtype == PPG_F32 || dtype == PPG_BF16 || dtype == PPG_F16; }
bool known_dim(int d) { return d == 32 || d == 64 || d == 128; }
bool known_block(int b) { return b == 32 || b == 64 || b == 128; }

int set_offsets(ppg_ctx* c, const char* who, int n_sets, const int32_t* off, const char* name, int* to) {
    if (!off) return fail(c, PPG_EINVAL, "%s: %s is NULL", who, name);
    for (int i = 0; i <= n_sets; i++) {
        if (off[i] < (i ? off[i - 1] : 0)) return fail(c, PPG_EINVAL, "%s: %s[%d] = %d descends or is negative", who, name, i, off[i]);
        to[i] = off[i];
    }
    return PPG_OK;
}
int set_count(ppg_ctx* c, const char* who, int n_sets) {
    if (n_sets < 0) return fail(c, PPG_EINVAL, "%s: n_sets is negative", who);
    if (n_sets > PPG_ATTN_MAX_SETS) return fail(c, PPG_ECAP, "%s: %d sets, at most %d per call", who, n_sets, PPG_ATTN_MAX_SETS);
    return PPG_OK;
}
// first block of every set; the blocks of 2^31 rows in blocks of 32 fit an int
void block_offsets(ppg::AttnSets& s, int block) {
    s.blk[0] = 0;
    for (int i = 0; i < s.n; i++) s.blk[i + 1] = s.blk[i] + (int)(((long long)s.k_off[i + 1] - s.k_off[i] + block - 1) / block);
    end_list(s, s.blk);
}

// what the kernels' launches cannot count
int too_large(ppg_ctx* c, const char* who) { return fail(c, PPG_ECAP, "%s: more rows or blocks than one launch holds (2^32 threads)", who); }

hipStream_t stream_of(ppg_ctx* c, void* stream) { return stream == PPG_STREAM_DEFAULT ? nullptr : stream ? (hipStream_t)stream : c->post; }
int finish(ppg_ctx* c, const char* who, hipError_t e, void* stream) {
    if (e == hipSuccess && !stream) e = hipStreamSynchronize(c->post);
    if (e != hipSuccess) return fail(c, PPG_EHIP, "%s: %s", who, hipGetErrorString(e));
    return PPG_OK;
}

// Everything ppg_attention checks before it touches the GPU; fills the launch structures.
int attention_checked(ppg_ctx* c, const ppg_attention_args* a, bool sizes_only, ppg::AttentionLaunch& l, ppg::AttnSets& sets) {
    static const char* who = "ppg_attention";
    if (!a) return fail(c, PPG_EINVAL, "%s: args is NULL", who);
    if (!known_type(a->dtype)) return fail(c, PPG_EINVAL, "%s: dtype %d is none of PPG_F32, PPG_BF16, PPG_F16", who, a->dtype);
    if (!known_dim(a->head_dim)) return fail(c, PPG_EINVAL, "%s: head_dim %d (32, 64 and 128 are built)", who, a->head_dim);
    if (!(a->scale > 0.f) || !(a->scale <= 1e37f)) return fail(c, PPG_EINVAL, "%s: scale must be positive, at most 1e37", who);
    int rc = set_count(c, who, a->n_sets);
    if (rc) return rc;
    sets.n = a->n_sets;
    if ((rc = set_offsets(c, who, a->n_sets, a->q_off, "q_off", sets.q_off))) return rc;
    if ((rc = set_offsets(c, who, a->n_sets, a->k_off, "k_off", sets.k_off))) return rc;
    const long long nq = (long long)sets.q_off[sets.n] - sets.q_off[0], nk = (long long)sets.k_off[sets.n] - sets.k_off[0];
    if (nq * a->q.heads >= kMostVectors || nk * a->k.heads >= kMostVectors)
        return fail(c, PPG_ECAP, "%s: rows times heads must stay below 2^31 - 2^10", who);
    if ((uintptr_t)a->lse % 4 || (uintptr_t)a->sel % 4) return fail(c, PPG_EINVAL, "%s: lse or sel is not at a multiple of 4", who);
    const ppg_rows* r[4] = {&a->q, &a->k, &a->v, &a->out};
    static const char* name[4] = {"q", "k", "v", "out"};
    for (int i = 0; i < 4; i++) {
        ppg_rows t = *r[i];
        if (sizes_only) t.p = (void*)16;
        const bool keys = i == 1 || i == 2;
        const char* fault = rows_fault(t, a->dtype, a->head_dim, keys ? nk : nq, i == 3);
        if (fault) return fail(c, PPG_EINVAL, "%s: %s: %s", who, name[i], fault);
    }
    if (a->k.heads != a->v.heads || a->q.heads != a->out.heads || a->q.heads % a->k.heads)
        return fail(c, PPG_EINVAL, "%s: heads of k and v, and of q and out, must agree, and the first divide the second", who);
    if (a->sel || a->n_sel || a->block) {
        if (!known_block(a->block)) return fail(c, PPG_EINVAL, "%s: block %d (32, 64 and 128 are built)", who, a->block);
        if (a->n_sel < 1) return fail(c, PPG_EINVAL, "%s: n_sel must be at least 1", who);
        if (a->n_sel > PPG_ATTN_MAX_SEL) return fail(c, PPG_ECAP, "%s: n_sel %d, at most %d", who, a->n_sel, PPG_ATTN_MAX_SEL);
        if (nq * a->q.heads * a->n_sel >= (1LL << 30)) return fail(c, PPG_ECAP, "%s: rows times heads times n_sel must stay below 2^30", who);
        if (!a->sel && !sizes_only && nq) return fail(c, PPG_EINVAL, "%s: block or n_sel is set and sel is NULL", who);
        block_offsets(sets, a->block);
    }
    l.scale = a->scale;
    l.q = a->q; l.k = a->k; l.v = a->v; l.out = a->out;
    l.skip = a->skip; l.lse = a->lse;
    l.block = a->block; l.n_sel = a->n_sel; l.sel = a->sel;
    l.work = a->work;
    return PPG_OK;
}

}  // namespace

extern "C" {

int ppg_resident_frame(ppg_ctx* c, int frame, const float** d_desc, const float** d_pos, int* n) {
    if (!c) return PPG_EINVAL;
    const float* desc = nullptr;
    int rows = 0;
    const int rc = ppg_ctx_last_desc(c, frame, &desc, &rows);
    if (rc) return rc;
    if (d_desc) *d_desc = desc;
    if (d_pos) *d_pos = c->slot[c->last_out_slot].kp_un + (size_t)frame * c->maxn * 2;
    if (n) *n = rows;
    return PPG_OK;
}

int ppg_rotary_frequencies(int n, double base, double scale, double extent, double low, double high, double* freq) {
    if (n < 0 || (n && !freq) || !(base > 0) || !(scale >= 1) || !std::isfinite(base) || !std::isfinite(scale))
        return fail(nullptr, PPG_EINVAL, "ppg_rotary_frequencies: n >= 0, base > 0 and scale >= 1 are needed");
    if (scale > 1 && (!(extent > 0) || !(low >= 0) || !(high > low) || !std::isfinite(extent) || !std::isfinite(high)))
        return fail(nullptr, PPG_EINVAL, "ppg_rotary_frequencies: with scale > 1, extent > 0 and high > low >= 0 are needed");
    for (int j = 0; j < n; j++) {
        const double f = std::pow(base, -(double)j / n);
        double keep = 1;   // how much of the unstretched frequency stays
        if (scale > 1) {
            const double turns = extent * f / 6.283185307179586476925;
            keep = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
        }
        freq[j] = f * (keep + (1 - keep) / scale);
    }
    return PPG_OK;
}

int ppg_rotary(ppg_ctx* c, const ppg_rotary_args* a, void* stream) {
    static const char* who = "ppg_rotary";
    if (!a) return fail(c, PPG_EINVAL, "%s: args is NULL", who);
    if (!known_type(a->dtype)) return fail(c, PPG_EINVAL, "%s: dtype %d is none of PPG_F32, PPG_BF16, PPG_F16", who, a->dtype);
    if (!known_dim(a->head_dim)) return fail(c, PPG_EINVAL, "%s: head_dim %d (32, 64 and 128 are built)", who, a->head_dim);
    if (a->layout != PPG_ROTARY_INTERLEAVED && a->layout != PPG_ROTARY_HALF) return fail(c, PPG_EINVAL, "%s: unknown layout %d", who, a->layout);
    if (a->n_axes != 1 && a->n_axes != 2) return fail(c, PPG_EINVAL, "%s: n_axes must be 1 or 2", who);
    if (a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % (2 * a->n_axes))
        return fail(c, PPG_EINVAL, "%s: rot_dim %d must be a multiple of %d, at most head_dim", who, a->rot_dim, 2 * a->n_axes);
    if (a->n_rows[0] < 0 || a->n_rows[1] < 0) return fail(c, PPG_EINVAL, "%s: n_rows is negative", who);
    if (a->rot_dim && (!a->freq || (uintptr_t)a->freq % 8) && (a->n_rows[0] || a->n_rows[1]))
        return fail(c, PPG_EINVAL, "%s: freq is NULL or not at a multiple of 8", who);
    ppg::RotaryLaunch l;
    l.head_dim = a->head_dim; l.rot_dim = a->rot_dim; l.layout = a->layout; l.inverse = a->inverse != 0; l.n_axes = a->n_axes;
    l.freq = a->freq;
    for (int i = 0; i < 2; i++) {
        l.n_rows[i] = a->n_rows[i];
        l.pos[i] = a->pos[i];
        l.src[i] = a->src[i];
        l.dst[i] = a->dst[i];
        if (!a->n_rows[i]) continue;
        if (a->rot_dim && (!a->pos[i] || (uintptr_t)a->pos[i] % 4)) return fail(c, PPG_EINVAL, "%s: pos[%d] is NULL or not at a multiple of 4", who, i);
        if ((long long)a->n_rows[i] * a->src[i].heads >= kMostVectors) return fail(c, PPG_ECAP, "%s: rows times heads must stay below 2^31 - 2^10", who);
        const char* fault = rows_fault(a->src[i], a->dtype, a->head_dim, a->n_rows[i], false);
        if (fault) return fail(c, PPG_EINVAL, "%s: src[%d]: %s", who, i, fault);
        if ((fault = rows_fault(a->dst[i], a->dtype, a->head_dim, a->n_rows[i], true))) return fail(c, PPG_EINVAL, "%s: dst[%d]: %s", who, i, fault);
        if (a->src[i].heads != a->dst[i].heads) return fail(c, PPG_EINVAL, "%s: src[%d] and dst[%d] differ in heads", who, i, i);
        if (a->src[i].p == a->dst[i].p && (a->src[i].row != a->dst[i].row || a->src[i].head != a->dst[i].head))
            return fail(c, PPG_EINVAL, "%s: dst[%d] is src[%d] with other strides", who, i, i);
    }
    if (!ppg::rotary_fits(l)) return too_large(c, who);
    if (!c) return fail(c, PPG_EINVAL, "%s: ctx is NULL", who);
    DeviceScope dev(c->cfg.device_id);
    HIPCHK(c, dev.err);
    return finish(c, who, ppg::launch_rotary(a->dtype, l, stream_of(c, stream)), stream);
}

int ppg_block_means(ppg_ctx* c, const ppg_block_means_args* a, void* stream) {
    static const char* who = "ppg_block_means";
    if (!a) return fail(c, PPG_EINVAL, "%s: args is NULL", who);
    if (!known_type(a->dtype)) return fail(c, PPG_EINVAL, "%s: dtype %d is none of PPG_F32, PPG_BF16, PPG_F16", who, a->dtype);
    if (!known_dim(a->head_dim)) return fail(c, PPG_EINVAL, "%s: head_dim %d (32, 64 and 128 are built)", who, a->head_dim);
    if (!known_block(a->block)) return fail(c, PPG_EINVAL, "%s: block %d (32, 64 and 128 are built)", who, a->block);
    int rc = set_count(c, who, a->n_sets);
    if (rc) return rc;
    ppg::AttnSets sets;
    sets.n = a->n_sets;
    if ((rc = set_offsets(c, who, a->n_sets, a->k_off, "k_off", sets.k_off))) return rc;
    const long long nk = (long long)sets.k_off[sets.n] - sets.k_off[0];
    const char* fault = rows_fault(a->k, a->dtype, a->head_dim, nk, false);
    if (fault) return fail(c, PPG_EINVAL, "%s: k: %s", who, fault);
    if (nk && (!a->mean || !a->count)) return fail(c, PPG_EINVAL, "%s: mean or count is NULL", who);
    if ((uintptr_t)a->mean % 16 || (uintptr_t)a->count % 4) return fail(c, PPG_EINVAL, "%s: mean is not at a multiple of 16, or count of 4", who);
    if (nk * a->k.heads >= kMostVectors) return fail(c, PPG_ECAP, "%s: rows times heads must stay below 2^31 - 2^10", who);
    block_offsets(sets, a->block);
    if (!ppg::block_means_fits(sets)) return too_large(c, who);
    ppg::BlockMeansLaunch l;
    l.block = a->block; l.k = a->k; l.skip = a->skip; l.mean = a->mean; l.count = a->count;
    if (!c) return fail(c, PPG_EINVAL, "%s: ctx is NULL", who);
    DeviceScope dev(c->cfg.device_id);
    HIPCHK(c, dev.err);
    return finish(c, who, ppg::launch_block_means(a->dtype, a->head_dim, l, sets, stream_of(c, stream)), stream);
}

int ppg_block_select(ppg_ctx* c, const ppg_block_select_args* a, void* stream) {
    static const char* who = "ppg_block_select";
    if (!a) return fail(c, PPG_EINVAL, "%s: args is NULL", who);
    if (!known_type(a->dtype)) return fail(c, PPG_EINVAL, "%s: dtype %d is none of PPG_F32, PPG_BF16, PPG_F16", who, a->dtype);
    if (!known_dim(a->head_dim)) return fail(c, PPG_EINVAL, "%s: head_dim %d (32, 64 and 128 are built)", who, a->head_dim);
    if (!known_block(a->block)) return fail(c, PPG_EINVAL, "%s: block %d (32, 64 and 128 are built)", who, a->block);
    if (a->n_sel < 1) return fail(c, PPG_EINVAL, "%s: n_sel must be at least 1", who);
    if (a->n_sel > PPG_ATTN_MAX_SEL) return fail(c, PPG_ECAP, "%s: n_sel %d, at most %d", who, a->n_sel, PPG_ATTN_MAX_SEL);
    int rc = set_count(c, who, a->n_sets);
    if (rc) return rc;
    ppg::AttnSets sets;
    sets.n = a->n_sets;
    if ((rc = set_offsets(c, who, a->n_sets, a->q_off, "q_off", sets.q_off))) return rc;
    if ((rc = set_offsets(c, who, a->n_sets, a->k_off, "k_off", sets.k_off))) return rc;
    const long long nq = (long long)sets.q_off[sets.n] - sets.q_off[0], nk = (long long)sets.k_off[sets.n] - sets.k_off[0];
    const char* fault = rows_fault(a->q, a->dtype, a->head_dim, nq, false);
    if (fault) return fail(c, PPG_EINVAL, "%s: q: %s", who, fault);
    if (a->kv_heads < 1 || a->q.heads % a->kv_heads) return fail(c, PPG_EINVAL, "%s: kv_heads must divide the heads of q", who);
    if ((nq && !a->sel) || (nq && nk && (!a->mean || !a->count))) return fail(c, PPG_EINVAL, "%s: sel, mean or count is NULL", who);
    if ((uintptr_t)a->mean % 16 || (uintptr_t)a->count % 4 || (uintptr_t)a->sel % 4)
        return fail(c, PPG_EINVAL, "%s: mean is not at a multiple of 16, or count or sel of 4", who);
    if (nq * a->q.heads >= kMostVectors || nk * a->kv_heads >= kMostVectors || nq * a->kv_heads * a->n_sel >= kMostVectors)
        return fail(c, PPG_ECAP, "%s: rows times heads (and times n_sel) must stay below 2^31 - 2^10", who);
    block_offsets(sets, a->block);
    ppg::BlockSelectLaunch l;
    l.block = a->block; l.kv_heads = a->kv_heads; l.n_sel = a->n_sel; l.q = a->q; l.mean = a->mean; l.count = a->count; l.sel = a->sel;
    if (!ppg::block_select_fits(l, sets)) return too_large(c, who);
    if (!c) return fail(c, PPG_EINVAL, "%s: ctx is NULL", who);
    DeviceScope dev(c->cfg.device_id);
    HIPCHK(c, dev.err);
    return finish(c, who, ppg::launch_block_select(a->dtype, a->head_dim, l, sets, stream_of(c, stream)), stream);
}

size_t ppg_attention_work(const ppg_attention_args* a) {
    ppg::AttentionLaunch l;
    ppg::AttnSets sets;
    if (!a || !a->q_off || !a->k_off || attention_checked(nullptr, a, true, l, sets)) return 0;
    const size_t need = ppg::attention_work(a->dtype, a->head_dim, l, sets);
    return need == ppg::kNoWork ? 0 : need;
}

int ppg_attention(ppg_ctx* c, const ppg_attention_args* a, void* stream) {
    ppg::AttentionLaunch l;
    ppg::AttnSets sets;
    const int rc = attention_checked(c, a, false, l, sets);
    if (rc) return rc;
    const size_t need = ppg::attention_work(a->dtype, a->head_dim, l, sets);
    if (need == ppg::kNoWork) return too_large(c, "ppg_attention");
    if (need && (!a->work || a->work_bytes < need || (uintptr_t)a->work % 256))
        return fail(c, PPG_EINVAL, "ppg_attention: work must be %zu bytes (ppg_attention_work), 256-byte aligned", need);
    if (!c) return fail(c, PPG_EINVAL, "ppg_attention: ctx is NULL");
    DeviceScope dev(c->cfg.device_id);
    HIPCHK(c, dev.err);
    return finish(c, "ppg_attention", ppg::launch_attention(a->dtype, a->head_dim, l, sets, stream_of(c, stream)), stream);
}

}  // extern "C"
