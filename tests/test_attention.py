"""Attention between descriptor sets: rotary positions, block means, block selection, attention over whole sets and over
selected blocks, against plain implementations in 64 bits; what the entry points refuse (no GPU needed).

Tolerances.  A rounding to a type is off by at most half a step, u = eps / 2 relative to the value.  For attention, with
n keys and D components: a product q.k in 32 bits is off by at most (D + 4) 2^-23 sum|q||k|, its exponent's argument by
2^-23 of itself; the weights therefore by a factor 1 + 4 E with E the largest of those (twice for numerator and
denominator, twice for the maximum that is subtracted).  Sums over the keys are taken in tiles of at least 32, so they add
at most (n / 32 + 64) roundings.  With 16-bit types a weight is rounded once (u of the type; below fp16's smallest normal
number 2^-25 absolutely, with a denominator of at least 1), and the result once more.  A stands for sum p |v|.  Selected
blocks with bf16: every block's mean passes through fp16, scaled, which is off by 2^-11 of its components and 2^-38 of its
largest (at most max |v|); the means' weights add up to 1, so that is 2^-11 A + 2^-38 max |v| more (max |v| <= sum |v|)."""
import ctypes as C
import math

import numpy as np
import pytest

TYPES = ("fp32", "bf16", "fp16")


def _u(dtype):
    return {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}[dtype]


# ------------------------------------------------------------------------------------------------ refusals, on the CPU

def _rows(pkg, heads=2, row=None, head=64, p=4096):
    return pkg.Rows(p, heads, heads * 64 if row is None else row, head)


def _attention(pkg, **kw):
    f = dict(dtype=pkg.BF16, head_dim=64, scale=0.125, q_off=pkg.offsets([0, 5]), k_off=pkg.offsets([0, 7]), q=_rows(pkg), k=_rows(pkg),
             v=_rows(pkg), out=_rows(pkg))
    f.update(kw)
    return pkg.attention_args(**f)


def _refusal(pkg, call, args):
    """(status, reason) of a call without a context: argument checks come first, the missing context last."""
    L = pkg.lib()
    rc = getattr(L, call)(None, args, None)
    return rc, L.ppg_last_error(None).decode()


def test_valid_arguments_are_refused_only_for_the_missing_context(pkg):
    assert _refusal(pkg, "ppg_attention", _attention(pkg)) == (pkg.PPG_EINVAL, "ppg_attention: ctx is NULL")
    for call in ("ppg_attention", "ppg_rotary", "ppg_block_means", "ppg_block_select"):
        rc, why = _refusal(pkg, call, None)
        assert rc == pkg.PPG_EINVAL and "args is NULL" in why
    assert pkg.lib().ppg_resident_frame(None, 0, None, None, None) == pkg.PPG_EINVAL


@pytest.mark.parametrize("change, code, word", [
    (dict(dtype=3), "PPG_EINVAL", "dtype"), (dict(head_dim=48), "PPG_EINVAL", "head_dim"), (dict(scale=0.0), "PPG_EINVAL", "scale"),
    (dict(scale=-1.0), "PPG_EINVAL", "scale"), (dict(scale=float("nan")), "PPG_EINVAL", "scale"), (dict(scale=float("inf")), "PPG_EINVAL", "scale"),
    (dict(q_off=[0, 5, 4], k_off=[0, 1, 2]), "PPG_EINVAL", "q_off[2]"), (dict(q_off=[-1, 5]), "PPG_EINVAL", "q_off[0]"),
    (dict(k_off=[3, 2]), "PPG_EINVAL", "k_off[1]"), (dict(q_off=list(range(130)), k_off=list(range(130))), "PPG_ECAP", "129 sets"),
    (dict(q="null"), "PPG_EINVAL", "q: address is NULL"), (dict(k=dict(p=4104)), "PPG_EINVAL", "k: address"),
    (dict(v=dict(row=132)), "PPG_EINVAL", "v: a stride"), (dict(k=dict(row=-128)), "PPG_EINVAL", "k: stride"),
    (dict(out=dict(row=64)), "PPG_EINVAL", "overlap"), (dict(out=dict(head=0)), "PPG_EINVAL", "overlap"),
    (dict(q=dict(heads=0)), "PPG_EINVAL", "heads"), (dict(k=dict(heads=1, row=64)), "PPG_EINVAL", "heads of k and v"),
    (dict(q=dict(heads=3, row=192), out=dict(heads=3, row=192)), "PPG_EINVAL", "divide"),
    (dict(block=48, n_sel=4, sel=4096), "PPG_EINVAL", "block 48"), (dict(block=64, n_sel=0, sel=4096), "PPG_EINVAL", "n_sel"),
    (dict(block=64, n_sel=65, sel=4096), "PPG_ECAP", "n_sel 65"), (dict(block=64, n_sel=4), "PPG_EINVAL", "sel is NULL"),
    (dict(sel=4096), "PPG_EINVAL", "block 0"), (dict(scale=2e37), "PPG_EINVAL", "scale"), (dict(lse=4098), "PPG_EINVAL", "lse"),
    (dict(block=64, n_sel=4, sel=4097), "PPG_EINVAL", "sel"), (dict(q_off=[0, 1 << 30]), "PPG_ECAP", "2^31"), (dict(k_off=[0, 2000000000]), "PPG_ECAP", "2^31"),
    (dict(q_off=[0, 1 << 24], block=64, n_sel=64, sel=4096), "PPG_ECAP", "2^30"),
])
def test_attention_refuses(pkg, change, code, word):
    kw = {}
    for k, x in change.items():
        kw[k] = _rows(pkg, p=None) if x == "null" else _rows(pkg, **x) if isinstance(x, dict) else pkg.offsets(x) if isinstance(x, list) else x
    rc, why = _refusal(pkg, "ppg_attention", _attention(pkg, **kw))
    assert rc == getattr(pkg, code) and word in why, (rc, why)


def test_attention_refuses_offsets_that_are_missing(pkg):
    a = _attention(pkg)
    a.k_off = None
    assert _refusal(pkg, "ppg_attention", a) == (pkg.PPG_EINVAL, "ppg_attention: k_off is NULL")
    assert pkg.lib().ppg_attention_work(a) == 0
    a = _attention(pkg)
    a.n_sets = -1
    assert "n_sets" in _refusal(pkg, "ppg_attention", a)[1]


@pytest.mark.parametrize("change, word", [
    (dict(dtype=-1), "dtype"), (dict(head_dim=96), "head_dim"), (dict(layout=2), "layout"), (dict(n_axes=3), "n_axes"),
    (dict(rot_dim=66), "rot_dim"), (dict(rot_dim=-2), "rot_dim"), (dict(rot_dim=30, n_axes=2), "rot_dim"), (dict(freq=None), "freq"),
    (dict(n_rows=(-1,)), "n_rows"), (dict(pos=(None,)), "pos[0]"), (dict(dst="overlap"), "other strides"), (dict(dst="heads"), "heads"),
    (dict(pos=(4098,)), "pos[0]"), (dict(freq=4100), "freq"), (dict(n_rows=((1 << 30),)), "2^31"),
])
def test_rotary_refuses(pkg, change, word):
    f = dict(dtype=pkg.F16, head_dim=64, rot_dim=64, layout=0, n_axes=1, freq=4096, n_rows=(3,), pos=(4096,), src=(_rows(pkg),),
             dst=(_rows(pkg, p=8192),))
    f.update({k: v for k, v in change.items() if k != "dst"})
    if change.get("dst") == "overlap":
        f["dst"] = (_rows(pkg, row=256),)
    if change.get("dst") == "heads":
        f["dst"] = (_rows(pkg, heads=4, p=8192),)
    rc, why = _refusal(pkg, "ppg_rotary", pkg.rotary_args(**f))
    assert rc == (pkg.PPG_ECAP if "2^" in word else pkg.PPG_EINVAL) and word in why, why


@pytest.mark.parametrize("change, code, word", [
    (dict(dtype=9), "PPG_EINVAL", "dtype"), (dict(head_dim=256), "PPG_EINVAL", "head_dim"), (dict(block=16), "PPG_EINVAL", "block"),
    (dict(mean=None), "PPG_EINVAL", "mean"), (dict(count=None), "PPG_EINVAL", "count"), (dict(mean=4100), "PPG_EINVAL", "mean"),
    (dict(k_off=[0, 4, 2]), "PPG_EINVAL", "k_off[2]"), (dict(k_off=list(range(200))), "PPG_ECAP", "sets"), (dict(k="null"), "PPG_EINVAL", "k: address"),
])
def test_block_means_refuses(pkg, change, code, word):
    f = dict(dtype=pkg.F32, head_dim=64, block=64, k_off=[0, 9], k=_rows(pkg), mean=4096, count=4096)
    f.update(change)
    f["k_off"] = pkg.offsets(f["k_off"])
    if f["k"] == "null":
        f["k"] = _rows(pkg, p=None)
    rc, why = _refusal(pkg, "ppg_block_means", pkg.block_means_args(**f))
    assert rc == getattr(pkg, code) and word in why, why


@pytest.mark.parametrize("change, code, word", [
    (dict(n_sel=0), "PPG_EINVAL", "n_sel"), (dict(n_sel=65), "PPG_ECAP", "n_sel"), (dict(kv_heads=3), "PPG_EINVAL", "kv_heads"),
    (dict(kv_heads=0), "PPG_EINVAL", "kv_heads"), (dict(sel=None), "PPG_EINVAL", "sel"), (dict(mean=None), "PPG_EINVAL", "mean"),
    (dict(block=0), "PPG_EINVAL", "block"), (dict(q_off=[1, 0]), "PPG_EINVAL", "q_off"), (dict(head_dim=0), "PPG_EINVAL", "head_dim"),
])
def test_block_select_refuses(pkg, change, code, word):
    f = dict(dtype=pkg.F32, head_dim=64, block=64, q_off=[0, 4], k_off=[0, 9], q=_rows(pkg), kv_heads=2, mean=4096, count=4096, n_sel=4, sel=4096)
    f.update(change)
    f["q_off"], f["k_off"] = pkg.offsets(f["q_off"]), pkg.offsets(f["k_off"])
    rc, why = _refusal(pkg, "ppg_block_select", pkg.block_select_args(**f))
    assert rc == getattr(pkg, code) and word in why, why


def test_what_one_launch_cannot_count_is_refused(pkg):
    """2^32 threads or more, and strides whose products pass 64 bits."""
    wide = dict(heads=65535, row=65535 * 64, head=64)
    cases = [("ppg_rotary", pkg.rotary_args(dtype=pkg.BF16, head_dim=64, rot_dim=64, layout=0, n_axes=1, freq=4096, n_rows=(1 << 28,), pos=(4096,), src=(_rows(pkg, heads=1),), dst=(_rows(pkg, heads=1, p=8192),))),
             ("ppg_block_means", pkg.block_means_args(dtype=pkg.F32, head_dim=64, block=32, k_off=pkg.offsets([0, 1 << 29]), k=_rows(pkg), mean=4096, count=4096)),
             ("ppg_block_select", pkg.block_select_args(dtype=pkg.F32, head_dim=64, block=64, q_off=pkg.offsets([0, 1 << 27]), k_off=pkg.offsets([0, 9]), q=_rows(pkg, heads=1),
                                                       kv_heads=1, mean=4096, count=4096, n_sel=4, sel=4096)),
             ("ppg_attention", _attention(pkg, q_off=pkg.offsets([0] + [32640 + i for i in range(128)]), k_off=pkg.offsets([0] * 129), **{x: _rows(pkg, **wide) for x in ("q", "k", "v", "out")})),
             ("ppg_attention", _attention(pkg, q_off=pkg.offsets([0, 16384]), k_off=pkg.offsets([0, 64]), block=32, n_sel=1, sel=4096, dtype=pkg.BF16, head_dim=32,
                                          q=_rows(pkg, **wide), out=_rows(pkg, **wide), k=_rows(pkg, heads=1), v=_rows(pkg, heads=1))),
             ("ppg_attention", _attention(pkg, q_off=pkg.offsets([0, 1 << 27]), block=64, n_sel=3, sel=4096))]
    for call, args in cases:
        rc, why = _refusal(pkg, call, args)
        assert rc == pkg.PPG_ECAP and "one launch" in why, (call, rc, why)
    assert pkg.lib().ppg_attention_work(cases[-1][1]) == 0 and pkg.lib().ppg_attention_work(cases[-2][1]) == 0
    # (2^23 rows at the rows' own distance would be 2^63 components away: the heads are not that far apart)
    rc, why = _refusal(pkg, "ppg_attention", _attention(pkg, q_off=pkg.offsets([0, 1 << 23]), out=_rows(pkg, row=1 << 40, head=1 << 40)))
    assert rc == pkg.PPG_EINVAL and "overlap" in why, (rc, why)


def test_rotary_frequencies(pkg):
    n, base = 32, 10000.0
    plain = pkg.rotary_frequencies(n, base)
    assert np.allclose(plain, base ** (-np.arange(n) / n), rtol=1e-14, atol=0)
    f = pkg.rotary_frequencies(n, base, scale=4.0, extent=1024.0, low=1.0, high=16.0)
    turns = 1024.0 * plain / (2 * math.pi)
    assert np.array_equal(f[turns >= 16], plain[turns >= 16]) and np.allclose(f[turns <= 1], plain[turns <= 1] / 4, rtol=1e-14, atol=0)
    mid = (turns > 1) & (turns < 16)
    t = (turns[mid] - 1) / 15
    assert mid.any() and np.allclose(f[mid], plain[mid] * (t + (1 - t) / 4), rtol=1e-13, atol=0)
    assert len(pkg.rotary_frequencies(0)) == 0
    for bad in (dict(base=0.0), dict(scale=0.5), dict(scale=2.0, extent=0.0), dict(scale=2.0, low=3.0, high=3.0), dict(base=float("nan"))):
        with pytest.raises(pkg.PPGError):
            pkg.rotary_frequencies(8, **bad)


# ----------------------------------------------------------------------------------------------------------- on the GPU

@pytest.fixture(scope="module")
def gpu(pkg):
    import torch
    ctx = pkg.Context(pkg.default_config(64, 64), matcher_only=True)
    yield pkg, ctx, torch
    ctx.close()


def _t(torch, dtype):
    return {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[dtype]


def _kind(pkg, dtype):
    return {"fp32": pkg.F32, "bf16": pkg.BF16, "fp16": pkg.F16}[dtype]


def _view(pkg, x):
    return pkg.Rows(x.data_ptr(), x.shape[1], x.stride(0), x.stride(1))


def _rand(torch, seed, *shape):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g)


def _rotary_ref(torch, x, pos, freq, rot, layout, axes, inverse):
    """(64-bit result, |x| + |y| of every pair at both of its components)"""
    x = x.double()
    y, size = x.clone(), torch.zeros_like(x)
    half = rot // 2
    for j in range(half):
        i0, i1 = (j, j + half) if layout == 1 else (2 * j, 2 * j + 1)
        a = pos[:, 1 if axes == 2 and j >= half // 2 else 0].double() * freq[j]
        a = -a if inverse else a
        c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
        u, v = x[..., i0], x[..., i1]
        y[..., i0], y[..., i1] = u * c - v * s, u * s + v * c
        size[..., i0] = size[..., i1] = u.abs() + v.abs()
    return y, size


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", (0, 1))
@pytest.mark.parametrize("dim, rot, axes", ((64, 64, 2), (32, 32, 1), (128, 124, 2), (64, 32, 1), (64, 6, 1), (32, 0, 1), (128, 128, 1)))
def test_rotary(gpu, dtype, layout, dim, rot, axes):
    """Both tensors of a call, odd row counts, strided input, in place; far positions on one axis.
    Tolerance: cos and sin to 2^-22 (rounding of the reduced angle, two sums of rounded terms), two products and a sum in 32
    bits (2^-23 of the pair), one rounding to the type."""
    pkg, ctx, torch = gpu
    t = _t(torch, dtype)
    freq = torch.from_numpy(pkg.rotary_frequencies(max(rot // 2, 1), 10000.0)).cuda()
    big = _rand(torch, 5, 133, 3, 2 * dim).to(t).cuda()
    q, k = big[:, :, dim:], _rand(torch, 6, 47, 1, dim).to(t).cuda()
    pos = [(_rand(torch, 7 + i, n, axes) * (3e5 if axes == 1 else 700)).cuda() for i, n in enumerate((133, 47))]
    for inverse in (0, 1):
        oq, ok = torch.full((133, 3, dim), 7.0, dtype=t, device="cuda"), torch.empty_like(k)
        args = dict(dtype=_kind(pkg, dtype), head_dim=dim, rot_dim=rot, layout=layout, inverse=inverse, n_axes=axes, freq=freq.data_ptr())
        ctx.rotary(pkg.rotary_args((133, 47), [p.data_ptr() for p in pos], (_view(pkg, q), _view(pkg, k)), (_view(pkg, oq), _view(pkg, ok)), **args), pkg.STREAM_DEFAULT)
        for x, y, p in ((q, oq, pos[0]), (k, ok, pos[1])):
            ref, size = _rotary_ref(torch, x.cpu(), p.cpu(), freq.cpu(), rot, layout, axes, inverse)
            tol = _u(dtype) * ref.abs() * 1.01 + size * 2.0 ** -21 + (2.0 ** -25 if dtype == "fp16" else 0)
            assert ((y.cpu().double() - ref).abs() <= tol).all()
            assert torch.equal(y[..., rot:].contiguous().cpu(), x[..., rot:].contiguous().cpu())
        # in place, one tensor: the same bits
        z = q.clone()
        ctx.rotary(pkg.rotary_args((133,), (pos[0].data_ptr(),), (_view(pkg, z),), (_view(pkg, z),), **args), pkg.STREAM_DEFAULT)
        assert torch.equal(z, oq)


@pytest.mark.gpu
def test_rotary_inverse_gives_the_input_back_and_is_the_gradient(gpu):
    """The turn is linear and orthogonal: <g, R x> = <R^-1 g, x>, and differences of R along a direction are R of it."""
    pkg, ctx, torch = gpu
    freq = torch.from_numpy(pkg.rotary_frequencies(32)).cuda()
    pos = (_rand(torch, 1, 65, 1) * 1000).cuda()
    x, g = _rand(torch, 2, 65, 2, 64).cuda(), _rand(torch, 3, 65, 2, 64).cuda()

    def turn(v, inverse):
        y = torch.empty_like(v)
        ctx.rotary(pkg.rotary_args((65,), (pos.data_ptr(),), (_view(pkg, v),), (_view(pkg, y),), dtype=pkg.F32, head_dim=64, rot_dim=64, layout=1,
                                   inverse=inverse, n_axes=1, freq=freq.data_ptr()), pkg.STREAM_DEFAULT)
        return y
    assert (turn(turn(x, 0), 1) - x).abs().max() <= 4 * 2.0 ** -21 * x.abs().max()
    lhs, rhs = (g.double() * turn(x, 0).double()).sum(), (turn(g, 1).double() * x.double()).sum()
    assert abs(lhs - rhs) <= 2.0 ** -20 * (g.double().abs() * x.double().abs()).sum() * 2
    d = (turn(x + 0.5 * g, 0).double() - turn(x - 0.5 * g, 0).double())
    assert (d - turn(g, 0).double()).abs().max() <= 2.0 ** -19 * float(x.abs().max() + g.abs().max())


def _means_ref(torch, k, off, block, skip):
    k = k.double()
    means, counts = [], []
    for a, b in zip(off, off[1:]):
        for i in range(a, b, block):
            j = min(b, i + block)
            keep = torch.ones(j - i, dtype=torch.bool) if skip is None else skip[i:j] == 0
            counts.append(int(keep.sum()))
            means.append(k[i:j][keep].sum(0) / max(1, counts[-1]))
    return torch.stack(means) if means else torch.zeros(0, k.shape[1], k.shape[2], dtype=torch.float64), counts


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block, dim, heads", ((32, 64, 4), (64, 32, 3), (128, 128, 1)))
def test_block_means(gpu, dtype, block, dim, heads):
    """Ragged and empty sets, a first row that is not 0, short last blocks, a block without keys, NaN in skipped rows; strided keys.
    The sum is exact in 64 bits up to 2^-52, so the mean is the reference rounded once."""
    pkg, ctx, torch = gpu
    off = [5, 5, 6, 6 + 2 * block, 7 + 5 * block, 7 + 5 * block + 31]
    big = _rand(torch, 11, off[-1] + 9, heads, 2 * dim).to(_t(torch, dtype))
    skip = (torch.rand(off[-1] + 9, generator=torch.Generator().manual_seed(3)) < 0.3).to(torch.uint8)
    skip[6:6 + block] = 1     # a whole block
    big[skip != 0] = float("nan")
    k = big.cuda()[:, :, dim:]
    for sk in (skip, None):
        kk = k if sk is not None else torch.nan_to_num(k, nan=0.25)
        view = kk if kk.stride(2) == 1 else kk.contiguous()
        nb = sum((b - a + block - 1) // block for a, b in zip(off, off[1:]))
        mean, count = torch.full((nb + 1, heads, dim), 9.0, device="cuda"), torch.full((nb + 1,), -9, dtype=torch.int32, device="cuda")
        sd = None if sk is None else sk.cuda()
        ctx.block_means(pkg.block_means_args(pkg.offsets(off), dtype=_kind(pkg, dtype), head_dim=dim, block=block, k=_view(pkg, view),
                                             skip=None if sd is None else sd.data_ptr(), mean=mean.data_ptr(), count=count.data_ptr()), pkg.STREAM_DEFAULT)
        ref, cnt = _means_ref(torch, view.cpu(), off, block, sk)
        assert count[:nb].tolist() == cnt and count[nb] == -9 and (mean[nb] == 9.0).all()
        assert ((mean[:nb].cpu().double() - ref).abs() <= 2.0 ** -24 * ref.abs() + 2.0 ** -45).all()


def _select_ref(q, mean, count, q_off, k_off, block, kv_heads, n_sel):
    """numpy: descending by (score, lower block first), NaN below every number, then ascending by block."""
    group = q.shape[1] // kv_heads
    out = np.full((q.shape[0], kv_heads, n_sel), -7, np.int32)
    first = 0
    for a, b, ka, kb in zip(q_off, q_off[1:], k_off, k_off[1:]):
        nb = (kb - ka + block - 1) // block
        for r in range(a, b):
            for g in range(kv_heads):
                with np.errstate(all="ignore"):
                    sc = mean[first:first + nb, g].astype(np.float64) @ q[r, g * group:(g + 1) * group].astype(np.float64).sum(0)
                live = [i for i in range(nb) if count[first + i] > 0]
                live.sort(key=lambda i: (np.isnan(sc[i]), -sc[i] if not np.isnan(sc[i]) else 0.0, i))
                pick = sorted(live[:n_sel])
                out[r, g] = pick + [-1] * (n_sel - len(pick))
        first += nb
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim, heads, kv_heads, n_sel, nk", ((64, 4, 4, 16, 5000), (32, 4, 1, 1, 3000), (128, 8, 2, 64, 9000), (64, 2, 2, 7, 130),
                                                             (32, 3, 1, 33, 33), (64, 2, 2, 16, 80000), (32, 2, 1, 64, 120000),
                                                             (128, 2, 1, 5, 34815)))
def test_block_select(gpu, dtype, dim, heads, kv_heads, n_sel, nk):
    """Ragged sets (one without keys, one without queries), dead blocks, exact ties (repeated and all-zero means), NaN means, a
    zero query, infinite queries; rows outside the sets stay."""
    pkg, ctx, torch = gpu
    block = 32
    q_off, k_off = [2, 12, 12, 30, 31], [0, nk, nk + 40, nk + 40, nk + 40 + 777]
    q = _rand(torch, 21, 40, heads, dim).to(_t(torch, dtype))
    q[3] = 0
    q[4, 0, 0] = float("inf")
    nb = [(b - a + block - 1) // block for a, b in zip(k_off, k_off[1:])]
    mean = _rand(torch, 22, sum(nb), kv_heads, dim)
    count = torch.full((sum(nb),), block, dtype=torch.int32)
    g = torch.Generator().manual_seed(5)
    if nb[0] > 8:
        mean[5] = mean[2]
        mean[nb[0] - 1] = mean[2]
        mean[1] = 0
        mean[3] = float("nan")
        count[torch.randperm(nb[0], generator=g)[: nb[0] // 5]] = 0
    qd, md, cd = q.cuda(), mean.cuda(), count.cuda()
    sel = torch.full((40, kv_heads, n_sel), -7, dtype=torch.int32, device="cuda")
    ctx.block_select(pkg.block_select_args(pkg.offsets(q_off), pkg.offsets(k_off), dtype=_kind(pkg, dtype), head_dim=dim, block=block, q=_view(pkg, qd),
                                           kv_heads=kv_heads, mean=md.data_ptr(), count=cd.data_ptr(), n_sel=n_sel, sel=sel.data_ptr()), pkg.STREAM_DEFAULT)
    ref = _select_ref(q.float().numpy(), mean.numpy(), count.numpy(), q_off, k_off, block, kv_heads, n_sel)
    assert np.array_equal(sel.cpu().numpy(), ref)


def _attend_ref(torch, q, k, v, scale, q_off, k_off, skip, sel=None, block=0, n_sel=0):
    """64 bits: (out, lse, tolerance without the type's roundings, sum p|v|, sum|v| of the keys attended) per row and head."""
    f = torch.float64
    nq, h, d = q.shape
    kvh = k.shape[1]
    out, lse = torch.zeros(nq, h, d, dtype=f), torch.full((nq, h), -math.inf, dtype=f)
    tol, a_abs, v_abs = torch.zeros(nq, h, d, dtype=f), torch.zeros(nq, h, d, dtype=f), torch.zeros(nq, h, d, dtype=f)
    ltol = torch.zeros(nq, h, dtype=f)
    for a, b, ka, kb in zip(q_off, q_off[1:], k_off, k_off[1:]):
        for hh in range(h):
            g = hh // (h // kvh)
            for r0, r1 in [(a, b)] if sel is None else [(r, r + 1) for r in range(a, b)]:
                if r1 == r0:
                    continue
                if sel is None:
                    idx = torch.arange(ka, kb)
                else:
                    nb = (kb - ka + block - 1) // block
                    idx = [torch.arange(ka + i * block, min(kb, ka + i * block + block)) for i in sel[r0, g].tolist() if 0 <= i < nb]
                    idx = torch.cat(idx) if idx else torch.zeros(0, dtype=torch.long)
                if skip is not None:
                    idx = idx[skip[idx] == 0]
                if len(idx) == 0:
                    continue
                qq, kk, vv = q[r0:r1, hh].to(f), k[idx, g].to(f), v[idx, g].to(f)
                z = qq @ kk.t() * scale
                m = z.amax(1, keepdim=True)
                dead = (m == -math.inf)[:, 0]
                p = torch.exp(z - m.masked_fill(m == -math.inf, 0.0))
                total = p.sum(1, keepdim=True)
                o = p @ vv / total.masked_fill(total == 0, 1.0)
                aa = p @ vv.abs() / total.masked_fill(total == 0, 1.0)
                e = 2.0 ** -23 * ((d + 4) * scale * (qq.abs() @ kk.abs().t()).amax(1) + 2 * z.abs().nan_to_num(0, 0, 0).amax(1))
                rel = 4 * e + 2 * (len(idx) / 32 + 64) * 2.0 ** -24
                out[r0:r1, hh] = o
                lse[r0:r1, hh] = torch.where(dead, torch.full_like(m[:, 0], -math.inf), (m + torch.log(total))[:, 0])
                ltol[r0:r1, hh] = rel + 2.0 ** -22 * lse[r0:r1, hh].abs().nan_to_num(0, 0, 0)
                tol[r0:r1, hh], a_abs[r0:r1, hh], v_abs[r0:r1, hh] = rel[:, None] * aa, aa, vv.abs().sum(0).expand(r1 - r0, d)
    return out, lse, tol, a_abs, v_abs, ltol


def _check_attend(torch, dtype, got, lse, ref, blocks=False):
    out, rl, tol, a_abs, v_abs, ltol = ref
    u = _u(dtype)
    t = tol + (0 if dtype == "fp32" else u * a_abs * 1.01) + u * out.abs() * 1.01
    if dtype == "fp16":
        t = t + 2.0 ** -25 * (v_abs + 1)
    if dtype == "fp32":
        t = t + 2.0 ** -126
    if dtype == "bf16" and blocks:
        t = t + 2.0 ** -11 * a_abs + 2.0 ** -38 * v_abs.amax(-1, keepdim=True)
    err = (got.cpu().double() - out).abs()
    ok = (err <= t) | (out.isnan() & got.cpu().isnan())
    assert ok.all(), (float((err / t.clamp(min=1e-300))[~ok].max()), int((~ok).sum()))
    if lse is not None:
        l = lse.cpu().double()
        assert torch.equal(l == -math.inf, rl == -math.inf) and torch.equal(l.isnan(), rl.isnan())
        fin = rl.isfinite()
        assert ((l - rl).abs()[fin] <= ltol[fin] + 2.0 ** -22).all()


def _run_attention(gpu, dtype, q, k, v, scale, q_off, k_off, skip=None, sel=None, block=0, out=None, lse=True, stream=None):
    pkg, ctx, torch = gpu
    out = torch.full(q.shape, 3.0, dtype=q.dtype, device="cuda") if out is None else out
    ls = torch.full(q.shape[:2], 3.0, device="cuda") if lse else None
    args = pkg.attention_args(pkg.offsets(q_off), pkg.offsets(k_off), dtype=_kind(pkg, dtype), head_dim=q.shape[2], scale=scale, q=_view(pkg, q),
                              k=_view(pkg, k), v=_view(pkg, v), out=_view(pkg, out), skip=None if skip is None else skip.data_ptr(),
                              lse=ls.data_ptr() if lse else None, block=block, n_sel=0 if sel is None else sel.shape[2],
                              sel=None if sel is None else sel.data_ptr())
    need = ctx.attention_work(args)
    work = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    work.fill_(0xA5)
    args.work, args.work_bytes = work.data_ptr(), need
    ctx.attention(args, pkg.STREAM_DEFAULT if stream is None else stream)
    assert (work[need:] == 0xA5).all()      # nothing behind the asked-for bytes is touched
    return out, ls


# (dim, heads, kv_heads, query lengths, key lengths, share of skipped keys): from one row to several tiles a side, odd sizes, sets
# without queries or keys, many sets, shared key heads, few queries against long sets
SHAPES = [
    (64, 4, 4, [1], [1], 0.0), (64, 1, 1, [1], [0], 0.0), (32, 2, 2, [0], [5], 0.0), (128, 2, 1, [3], [64], 0.0), (64, 4, 4, [31, 0, 33, 1], [65, 7, 0, 1], 0.0),
    (64, 4, 4, [32], [63], 0.5), (32, 8, 8, [129, 64], [127, 128], 0.0), (128, 2, 2, [130, 257], [200, 33], 0.1), (64, 8, 2, [100, 5], [321, 1], 0.05),
    (64, 6, 2, [37], [500], 0.0), (64, 16, 1, [1], [3001], 0.05), (128, 8, 8, [1, 1], [2500, 1300], 0.0), (64, 4, 4, [500], [487], 0.0),
    (32, 1, 1, [700], [1025], 0.2), (64, 2, 2, [3] * 40, list(range(0, 160, 4)), 0.1), (64, 4, 1, [2], [20000], 0.9), (128, 5, 5, [64], [777], 1.0),
    (64, 1, 1, [1030], [2050], 0.03), (64, 4, 4, [257] * 9, [255] * 9, 0.03),
    # enough rows for the kernel that shares tiles between 128 of them: more keys than its mask window, every tail, shared key heads
    (64, 2, 2, [130] + [129] * 127, [4500] + [40] * 127, 0.05), (128, 2, 2, [130] + [129] * 127, [4500] + list(range(127)), 0.3),
    (32, 4, 4, [100, 129, 1, 0] * 32, [65, 0, 127, 3] * 31 + [64, 63, 8200, 1], 0.0), (64, 12, 4, [90, 129] * 20, [33, 64] * 20, 0.5),
    (128, 8, 2, [300] * 22, [130, 1] * 11, 0.0),
    # fewer rows against long sets: the same kernel with the keys in shares (the mask's window starts anywhere), rows of several tiles
    (64, 4, 4, [300], [9001], 0.05), (128, 4, 4, [140, 70], [9000, 300], 0.5), (32, 8, 8, [129], [5001], 0.0), (64, 8, 2, [9], [30011], 0.02),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "d%d_h%d_%d_q%d_k%d_n%d" % (s[0], s[1], s[2], sum(s[3]), sum(s[4]), len(s[3])))
def test_attention_whole_sets(gpu, dtype, shape):
    """Every length from none to several tiles, with rows in front of and behind the sets that must stay; skipped keys hold NaN and
    infinities."""
    pkg, ctx, torch = gpu
    dim, heads, kvh, ql, kl, share = shape
    q_off, k_off = np.cumsum([2] + ql).tolist(), np.cumsum([1] + kl).tolist()
    t = _t(torch, dtype)
    q, k, v = (1.5 * _rand(torch, 31, q_off[-1] + 3, heads, dim)).to(t), _rand(torch, 32, k_off[-1] + 2, kvh, dim).to(t), _rand(torch, 33, k_off[-1] + 2, kvh, dim).to(t)
    skip = None
    if share:
        skip = (torch.rand(k_off[-1] + 2, generator=torch.Generator().manual_seed(7)) < share).to(torch.uint8)
        gone = skip != 0
        k[gone], v[gone] = float("nan"), float("inf")
    scale = 1 / math.sqrt(dim)
    ref = _attend_ref(torch, q, k, v, scale, q_off, k_off, skip)
    out, lse = _run_attention(gpu, dtype, q.cuda(), k.cuda(), v.cuda(), scale, q_off, k_off, None if skip is None else skip.cuda())
    a, b = q_off[0], q_off[-1]
    assert (out[:a] == 3).all() and (out[b:] == 3).all() and (lse[:a] == 3).all() and (lse[b:] == 3).all()
    _check_attend(torch, dtype, out[a:b], lse[a:b], [x[a:b] for x in ref])
    out, _ = _run_attention(gpu, dtype, q.cuda(), k.cuda(), v.cuda(), scale, q_off, k_off, None if skip is None else skip.cuda(), lse=False)
    assert (out[:a] == 3).all() and (out[b:] == 3).all()
    _check_attend(torch, dtype, out[a:b], None, [x[a:b] for x in ref])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_strides(gpu, dtype):
    """Queries, keys and values as slices of one packed projection; heads outermost; keys shared by stride 0; output into a slice."""
    pkg, ctx, torch = gpu
    t = _t(torch, dtype)
    packed = _rand(torch, 41, 150, 3, 4, 64).to(t).cuda()
    q, k, v = packed[:, 0], packed[:, 1], packed[:, 2]
    home = torch.full((150, 2, 4, 64), 3.0, dtype=t, device="cuda")
    ref = _attend_ref(torch, q.cpu(), k.cpu(), v.cpu(), 0.125, [0, 70, 150], [0, 90, 150], None)
    out, lse = _run_attention(gpu, dtype, q, k, v, 0.125, [0, 70, 150], [0, 90, 150], out=home[:, 1])
    _check_attend(torch, dtype, out, lse, ref)
    assert (home[:, 0] == 3).all()
    qh, kh, vh = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    oh = torch.empty(4, 150, 64, dtype=t, device="cuda").transpose(0, 1)
    _run_attention(gpu, dtype, qh, kh, vh, 0.125, [0, 70, 150], [0, 90, 150], out=oh)
    assert torch.equal(oh.contiguous(), out.contiguous())
    k1, v1 = k[:, :1].expand(150, 4, 64), v[:, :1].expand(150, 4, 64)     # one key head seen as four
    ref = _attend_ref(torch, q.cpu(), k1.cpu(), v1.cpu(), 0.125, [0, 70, 150], [0, 90, 150], None)
    out, lse = _run_attention(gpu, dtype, q, k1, v1, 0.125, [0, 70, 150], [0, 90, 150])
    _check_attend(torch, dtype, out, lse, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", (3, 200))
def test_attention_extreme_values(gpu, dtype, rows):
    """Products that grow along the keys (the running maximum moves in every tile), that are all far below zero, -inf or NaN."""
    pkg, ctx, torch = gpu
    t = _t(torch, dtype)
    n = 700
    q, v = torch.zeros(rows, 1, 64), _rand(torch, 51, n, 1, 64)
    k = torch.zeros(n, 1, 64)
    q[:, 0, 0] = 1
    k[:, 0, 0] = torch.arange(n) * 0.25 - 90       # up to +85, exact in every type used
    k[:, 0, 0] = k[:, 0, 0].to(t).float()
    for case in ("up", "down", "low", "inf", "nan"):
        kk, qq = k.clone(), q.clone()
        if case == "down":
            kk = kk.flip(0)
        elif case == "low":
            kk[:, 0, 0] = -30000.0
        elif case == "inf":
            kk[:, 0, 0] = -math.inf
        elif case == "nan":
            qq[rows // 2] = float("nan")
        a, b, c = qq.to(t), kk.to(t), v.to(t)
        ref = _attend_ref(torch, a, b, c, 1.0, [0, rows], [0, n], None)
        if case == "inf":      # 0 * -inf of the other components is NaN: keep them out of the row
            b[:, 0, 1:] = 0
            a[:, 0, 1:] = 0
            ref[0][:], ref[1][:] = 0, -math.inf
            for x in ref[2:]:
                x.nan_to_num_(0, 0, 0)
        out, lse = _run_attention(gpu, dtype, a.cuda(), b.cuda(), c.cuda(), 1.0, [0, rows], [0, n])
        _check_attend(torch, dtype, out, lse, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ("bf16", "fp32"))
def test_attention_offsets_beyond_32_bits(gpu, dtype):
    """Row strides that put the last rows more than 2^31 components (and 2^32 bytes) behind the first."""
    pkg, ctx, torch = gpu
    t = _t(torch, dtype)
    n, stride = 70, (1 << 26) // (2 if dtype == "fp32" else 1)
    size = n * stride
    flat = torch.zeros(size, dtype=t, device="cuda")
    assert size > 1 << 31
    k = flat.as_strided((n, 2, 64), (stride, 128, 1))
    v = flat.as_strided((n, 2, 64), (stride, 128, 1), 64)
    src_k, src_v, q = _rand(torch, 61, n, 2, 64).to(t), _rand(torch, 62, n, 2, 64).to(t), _rand(torch, 63, 40, 4, 64).to(t)
    k.copy_(src_k)
    v.copy_(src_v)
    ref = _attend_ref(torch, q, src_k, src_v, 0.125, [0, 40], [0, n], None)
    out, lse = _run_attention(gpu, dtype, q.cuda(), k, v, 0.125, [0, 40], [0, n])
    _check_attend(torch, dtype, out, lse, ref)
    sel = torch.tensor([[[0, 1, 2], [2, 1, -1]]], dtype=torch.int32).repeat(40, 1, 1)
    ref = _attend_ref(torch, q, src_k, src_v, 0.125, [0, 40], [0, n], None, sel, 32, 3)
    out, lse = _run_attention(gpu, dtype, q.cuda(), k, v, 0.125, [0, 40], [0, n], sel=sel.cuda(), block=32)
    _check_attend(torch, dtype, out, lse, ref)
    mean, count = torch.empty(3, 2, 64, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    ctx.block_means(pkg.block_means_args(pkg.offsets([0, n]), dtype=_kind(pkg, dtype), head_dim=64, block=32, k=_view(pkg, k), mean=mean.data_ptr(),
                                         count=count.data_ptr()), pkg.STREAM_DEFAULT)
    assert ((mean.cpu().double() - _means_ref(torch, src_k, [0, n], 32, None)[0]).abs() <= 2.0 ** -23).all()


# (dim, heads, kv_heads, block, n_sel, query lengths, key lengths, skipped): one query, a few, many that crowd on few blocks or spread
BLOCK_SHAPES = [
    (64, 4, 4, 64, 16, [1], [5000], 0.0), (64, 4, 4, 64, 1, [3], [10], 0.0), (32, 8, 2, 32, 7, [5, 0, 3], [300, 40, 0], 0.1), (128, 2, 2, 128, 33, [17], [9000], 0.05),
    (64, 4, 4, 64, 16, [300, 211], [3000, 65], 0.05), (64, 8, 1, 32, 5, [90], [640], 0.5), (128, 4, 2, 64, 64, [33], [4100], 0.0), (32, 2, 2, 128, 3, [400], [1000], 0.0),
    (64, 3, 1, 64, 4, [50], [700], 1.0), (64, 32, 2, 64, 4, [70], [1000], 0.1), (64, 4, 4, 64, 16, [700], [8000], 0.0),
    # many entries on one to five blocks, groups of more than 32 heads, more entries and more blocks than a work-group holds at a time
    (64, 4, 4, 128, 5, [1000, 999, 998, 997, 996], [30, 200, 300, 500, 640], 0.05), (32, 40, 1, 128, 16, [260], [5000], 0.0), (32, 40, 1, 64, 3, [3], [500], 0.1),
    (64, 1, 1, 64, 16, [1100], [5000], 0.05), (128, 1, 1, 32, 16, [300], [300000], 0.0),
    # many sets of few rows or none: several in the rows that one work-group joins
    (64, 4, 2, 64, 6, [(7 * i) % 12 * (i % 5 > 0) for i in range(128)], [(37 * i) % 700 for i in range(128)], 0.05),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", BLOCK_SHAPES, ids=lambda s: "d%d_h%d_%d_b%d_n%d_q%d_k%d" % (s[0], s[1], s[2], s[3], s[4], sum(s[5]), sum(s[6])))
def test_attention_selected_blocks(gpu, dtype, shape):
    """Lists with gaps, numbers that name no block, a block listed twice, empty lists, crowds on one block; short last blocks;
    the result does not depend on the lists' order beyond rounding."""
    pkg, ctx, torch = gpu
    dim, heads, kvh, block, n_sel, ql, kl, share = shape
    q_off, k_off = np.cumsum([2] + ql).tolist(), np.cumsum([1] + kl).tolist()
    t = _t(torch, dtype)
    nq = q_off[-1] + 3
    q, k, v = _rand(torch, 71, nq, heads, dim).to(t), _rand(torch, 72, k_off[-1] + 2, kvh, dim).to(t), _rand(torch, 73, k_off[-1] + 2, kvh, dim).to(t)
    g = torch.Generator().manual_seed(9)
    sel = torch.full((nq, kvh, n_sel), 0x40000000, dtype=torch.int32)
    for a, b, ka, kb in zip(q_off, q_off[1:], k_off, k_off[1:]):
        nb = (kb - ka + block - 1) // block
        for r in range(a, b):
            for h in range(kvh):
                p = torch.randperm(nb, generator=g)[:n_sel].tolist()
                p = (p + [-1, nb, -5, 1 << 30] * 17)[:n_sel]
                if r % 5 == 1:
                    p = [-1] * n_sel                  # nothing
                elif r % 5 == 2 and n_sel > 1 and nb:
                    p[0] = p[1]                       # twice the same
                elif r % 5 == 3 and nb:
                    p[0] = nb - 1                     # a crowd on the last, short block
                sel[r, h] = torch.tensor(p, dtype=torch.int32)
    skip = None
    if share:
        skip = (torch.rand(k_off[-1] + 2, generator=g) < share).to(torch.uint8)
        gone = skip != 0
        k[gone], v[gone] = float("nan"), float("inf")
    scale = 1 / math.sqrt(dim)
    ref = _attend_ref(torch, q, k, v, scale, q_off, k_off, skip, sel, block, n_sel)
    out, lse = _run_attention(gpu, dtype, q.cuda(), k.cuda(), v.cuda(), scale, q_off, k_off, None if skip is None else skip.cuda(), sel.cuda(), block)
    a, b = q_off[0], q_off[-1]
    assert (out[:a] == 3).all() and (out[b:] == 3).all() and (lse[:a] == 3).all() and (lse[b:] == 3).all()
    _check_attend(torch, dtype, out[a:b], lse[a:b], [x[a:b] for x in ref], blocks=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ("bf16", "fp32"))
def test_selected_blocks_with_values_of_every_size(gpu, dtype):
    """Values from 1e-30 to 1e30 (a size per block and per component), infinities and NaN among the keys attended to: what is
    not finite stays in its component, the others keep their precision."""
    pkg, ctx, torch = gpu
    t = _t(torch, dtype)
    g = torch.Generator().manual_seed(12)
    q, k, v = _rand(torch, 74, 200, 2, 64).to(t), _rand(torch, 75, 1280, 2, 64).to(t), _rand(torch, 76, 1280, 2, 64)
    v = v * 10.0 ** torch.randint(-30, 31, (20, 1, 1), generator=g).repeat_interleave(64, 0) * 10.0 ** (-torch.arange(64) / 16.0)
    v[70, 0, 3], v[200, 1, 5], v[300, 0, 7] = math.inf, -math.inf, math.nan
    v = v.to(t)
    sel = torch.stack([torch.randperm(20, generator=g)[:5] for _ in range(400)]).view(200, 2, 5).to(torch.int32)
    ref = _attend_ref(torch, q, k, v, 0.125, [0, 200], [0, 1280], None, sel, 64, 5)
    out, lse = _run_attention(gpu, dtype, q.cuda(), k.cuda(), v.cuda(), 0.125, [0, 200], [0, 1280], sel=sel.cuda(), block=64)
    got, want = out.cpu().double(), ref[0]
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()) and want.isinf().any() and want.isnan().any()
    fin = want.isfinite()
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()])
    part = 0 if dtype == "fp32" else 2.0 ** -11 * ref[3] + 2.0 ** -38 * ref[3].nan_to_num(0, 0, 0).amax(-1, keepdim=True)
    tol = ref[2] + (0 if dtype == "fp32" else _u(dtype) * ref[3] * 1.01) + _u(dtype) * want.abs() * 1.01 + part + 2.0 ** -126
    assert ((got - want).abs()[fin] <= tol[fin]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_repeated_calls_give_the_same_bits(gpu, dtype):
    pkg, ctx, torch = gpu
    t = _t(torch, dtype)
    q, k, v = _rand(torch, 81, 600, 4, 64).to(t).cuda(), _rand(torch, 82, 6000, 2, 64).to(t).cuda(), _rand(torch, 83, 6000, 2, 64).to(t).cuda()
    sel = torch.randint(0, 94, (600, 2, 12), generator=torch.Generator().manual_seed(2), dtype=torch.int32).cuda()
    for kw in (dict(), dict(sel=sel, block=64)):
        first = _run_attention(gpu, dtype, q, k, v, 0.125, [0, 250, 600], [0, 3000, 6000], **kw)
        for _ in range(4):
            again = _run_attention(gpu, dtype, q, k, v, 0.125, [0, 250, 600], [0, 3000, 6000], **kw)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.gpu
def test_work_that_is_missing_or_small_is_refused(gpu):
    pkg, ctx, torch = gpu
    q, k = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(200000, 4, 64, dtype=torch.bfloat16, device="cuda")
    args = pkg.attention_args(pkg.offsets([0, 1]), pkg.offsets([0, 200000]), dtype=pkg.BF16, head_dim=64, scale=1.0, q=_view(pkg, q), k=_view(pkg, k),
                              v=_view(pkg, k), out=_view(pkg, q))
    need = ctx.attention_work(args)
    work = torch.empty(need + 512, dtype=torch.uint8, device="cuda")
    if need:
        for p, n in ((None, need), (work.data_ptr(), need - 1), (work.data_ptr() + 16, need)):
            args.work, args.work_bytes = p, n
            with pytest.raises(pkg.PPGError, match="work must be"):
                ctx.attention(args, pkg.STREAM_DEFAULT)


class _Chain:
    """What a matcher layer over a map does: positions on queries and keys, block means, selection, attention over the blocks, and
    attention between the frame's own points; buffers of its own."""

    def __init__(self, gpu, seed, dtype="bf16"):
        pkg, ctx, torch = gpu
        self.gpu, t = gpu, _t(torch, dtype)
        nq, nk = 300, 5000
        self.q_off, self.k_off = [0, 120, 300], [0, 2100, 5000]
        self.q, self.k, self.v = (torch.empty(n, 4, 64, dtype=t, device="cuda") for n in (nq, nk, nk))
        self.pos = [torch.rand(n, 2, device="cuda") * 640 for n in (nq, nk)]
        self.freq = torch.from_numpy(np.tile(pkg.rotary_frequencies(16, 640.0), 2)).cuda()
        self.fill(seed)
        self.rq, self.rk = torch.empty_like(self.q), torch.empty_like(self.k)
        nb = sum((b - a + 63) // 64 for a, b in zip(self.k_off, self.k_off[1:]))
        self.mean, self.count = torch.empty(nb, 4, 64, device="cuda"), torch.empty(nb, dtype=torch.int32, device="cuda")
        self.sel = torch.empty(nq, 4, 8, dtype=torch.int32, device="cuda")
        self.out, self.own = torch.empty_like(self.q), torch.empty_like(self.q)
        kind, qo, ko = _kind(pkg, dtype), pkg.offsets(self.q_off), pkg.offsets(self.k_off)
        V = lambda x: _view(pkg, x)  # noqa: E731
        self.rot = pkg.rotary_args((nq, nk), [p.data_ptr() for p in self.pos], (V(self.q), V(self.k)), (V(self.rq), V(self.rk)), dtype=kind, head_dim=64,
                                   rot_dim=64, layout=0, n_axes=2, freq=self.freq.data_ptr())
        self.means = pkg.block_means_args(ko, dtype=kind, head_dim=64, block=64, k=V(self.rk), mean=self.mean.data_ptr(), count=self.count.data_ptr())
        self.select = pkg.block_select_args(qo, ko, dtype=kind, head_dim=64, block=64, q=V(self.rq), kv_heads=4, mean=self.mean.data_ptr(),
                                            count=self.count.data_ptr(), n_sel=8, sel=self.sel.data_ptr())
        self.cross = pkg.attention_args(qo, ko, dtype=kind, head_dim=64, scale=0.125, q=V(self.rq), k=V(self.rk), v=V(self.v), out=V(self.out), block=64,
                                        n_sel=8, sel=self.sel.data_ptr())
        self.self_ = pkg.attention_args(qo, qo, dtype=kind, head_dim=64, scale=0.125, q=V(self.rq), k=V(self.rq), v=V(self.out), out=V(self.own))
        self.work = []
        for a in (self.cross, self.self_):
            n = ctx.attention_work(a)
            self.work.append(torch.empty(max(n, 1), dtype=torch.uint8, device="cuda"))
            a.work, a.work_bytes = self.work[-1].data_ptr(), n

    def fill(self, seed):
        pkg, ctx, torch = self.gpu
        for i, x in enumerate((self.q, self.k, self.v)):
            x.copy_(_rand(torch, 100 * seed + i, *x.shape))

    def run(self, stream, ctx=None):
        ctx = ctx or self.gpu[1]
        ctx.rotary(self.rot, stream)
        ctx.block_means(self.means, stream)
        ctx.block_select(self.select, stream)
        ctx.attention(self.cross, stream)
        ctx.attention(self.self_, stream)

    def check(self):
        pkg, ctx, torch = self.gpu
        for x, y, p in ((self.q, self.rq, self.pos[0]), (self.k, self.rk, self.pos[1])):
            ref, size = _rotary_ref(torch, x.cpu(), p.cpu(), self.freq.cpu(), 64, 0, 2, 0)
            assert ((y.cpu().double() - ref).abs() <= _u("bf16") * 1.01 * ref.abs() + size * 2.0 ** -21).all()
        sel = self.sel.cpu()
        assert np.array_equal(sel.numpy(), _select_ref(self.rq.cpu().float().numpy(), self.mean.cpu().numpy(), self.count.cpu().numpy(), self.q_off,
                                                       self.k_off, 64, 4, 8))
        rq, rk, v, out = (x.cpu() for x in (self.rq, self.rk, self.v, self.out))
        _check_attend(torch, "bf16", self.out, None, _attend_ref(torch, rq, rk, v, 0.125, self.q_off, self.k_off, None, sel, 64, 8), blocks=True)
        _check_attend(torch, "bf16", self.own, None, _attend_ref(torch, rq, rq, out, 0.125, self.q_off, self.q_off, None))

    def results(self):
        return [x.clone() for x in (self.rq, self.rk, self.mean, self.sel, self.out, self.own)]


@pytest.mark.gpu
def test_chain_on_the_contexts_stream_and_on_a_callers(gpu):
    """The operators one after another, each reading what the one before wrote: blocking calls on the context's stream, and a
    caller's stream without a wait in between; the same bits."""
    pkg, ctx, torch = gpu
    c = _Chain(gpu, 1)
    torch.cuda.synchronize()
    c.run(None)                      # returns with the results in place
    c.check()
    want = c.results()
    for x in (c.rq, c.rk, c.mean, c.sel, c.out, c.own):
        x.zero_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c.run(s.cuda_stream)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, c.results()))
    before = torch.cuda.current_device()
    c.run(pkg.STREAM_DEFAULT)
    torch.cuda.synchronize()
    assert torch.cuda.current_device() == before and all(torch.equal(a, b) for a, b in zip(want, c.results()))


@pytest.mark.gpu
def test_chain_captured_and_replayed(gpu):
    """Two captured chains, replayed with new inputs and with eager work between the replays: each replay equals the eager result."""
    pkg, ctx, torch = gpu
    chains = [_Chain(gpu, 1), _Chain(gpu, 2)]
    graphs = []
    for c in chains:
        g = torch.cuda.CUDAGraph()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=s):
            c.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for seed in range(3, 7):
        for i, c in enumerate(chains):
            c.fill(10 * seed + i)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for g, s in zip(graphs, streams):     # side by side: each chain has its own work
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        got = [c.results() for c in chains]
        for c, r in zip(chains, got):
            for x in (c.rq, c.rk, c.mean, c.sel, c.out, c.own):
                x.zero_()
            c.run(pkg.STREAM_DEFAULT)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(r, c.results()))


@pytest.mark.gpu
def test_two_contexts_on_two_threads(gpu):
    import threading
    pkg, ctx, torch = gpu
    chains = [_Chain(gpu, 5), _Chain(gpu, 6)]
    ctxs = [pkg.Context(pkg.default_config(64, 64), matcher_only=True) for _ in chains]
    torch.cuda.synchronize()
    want = []
    for c in chains:
        c.run(None)
        want.append(c.results())
    torch.cuda.synchronize()
    errors = []

    def worker(i):
        try:
            s = torch.cuda.Stream()
            for rep in range(10):
                chains[i].run(s.cuda_stream if rep % 2 else None, ctxs[i])
                s.synchronize()
                with torch.cuda.stream(s):
                    same = all(torch.equal(a, b) for a, b in zip(want[i], (chains[i].rq, chains[i].rk, chains[i].mean, chains[i].sel, chains[i].out, chains[i].own)))
                if not same:
                    errors.append((i, rep))
        except Exception as e:  # noqa: BLE001
            errors.append((i, repr(e)))
    ts = [threading.Thread(target=worker, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join(timeout=100)
    assert not errors and not any(t.is_alive() for t in ts)
    for c in ctxs:
        c.close()


@pytest.mark.gpu
def test_attention_between_resident_frames(gpu, synth):
    """A frame's descriptors against the next frame's, read where the extractor left them: 4 heads of 64, positions on two axes."""
    pkg, _, torch = gpu
    W, H = 128, 96
    ctx = pkg.Context(pkg.default_config(W, H, max_batch=2))
    with pytest.raises(pkg.PPGError, match="no extracted batch"):
        ctx.resident_frame(0)
    frames = ctx.extract_batch([synth.make_frame(H, W, 1, i, "sparse") for i in range(2)])
    with pytest.raises(pkg.PPGError, match="outside"):
        ctx.resident_frame(2)
    place = [ctx.resident_frame(i) for i in range(2)]
    assert [p[2] for p in place] == [f["n"] for f in frames] and min(f["n"] for f in frames) > 8
    desc = [torch.from_numpy(f["desc"]).view(-1, 4, 64) for f in frames]
    freq = torch.from_numpy(np.tile(pkg.rotary_frequencies(16, 640.0), 2)).cuda()
    turned = [torch.empty(f["n"], 4, 64, device="cuda") for f in frames]
    ctx.rotary(pkg.rotary_args([p[2] for p in place], [p[1] for p in place], [pkg.Rows(p[0], 4, 256, 64) for p in place], [_view(pkg, x) for x in turned],
                               dtype=pkg.F32, head_dim=64, rot_dim=64, layout=0, n_axes=2, freq=freq.data_ptr()))
    for f, d, x in zip(frames, desc, turned):
        ref, size = _rotary_ref(torch, d, torch.from_numpy(f["un"]), freq.cpu(), 64, 0, 2, 0)
        assert ((x.cpu().double() - ref).abs() <= 2.0 ** -24 * ref.abs() + size * 2.0 ** -21).all()
    out = torch.empty_like(turned[0])
    args = pkg.attention_args(pkg.offsets([0, place[0][2]]), pkg.offsets([0, place[1][2]]), dtype=pkg.F32, head_dim=64, scale=16.0, q=_view(pkg, turned[0]),
                              k=_view(pkg, turned[1]), v=pkg.Rows(place[1][0], 4, 256, 64), out=_view(pkg, out))
    need = ctx.attention_work(args)
    work = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    args.work, args.work_bytes = work.data_ptr(), need
    ctx.attention(args)
    ref = _attend_ref(torch, turned[0].cpu(), turned[1].cpu(), desc[1], 16.0, [0, place[0][2]], [0, place[1][2]], None)
    _check_attend(torch, "fp32", out, None, ref)
    ctx.close()
