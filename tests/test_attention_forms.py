"""Attention between descriptor sets where the sizes, layouts and values of test_attention.py do not lead: vectors so short that
their squares vanish, products far from zero, sums that cancel, and the forms of the kernels that only large or strided calls take.

References are in 64 bits; tolerances are those of test_attention.py unless a test derives its own.  (The room that those leave for
block means in fp16 is not needed any more: what passes between two kernels of a call is in 32 bits.)"""
import math

import numpy as np
import pytest

from test_attention import TYPES, _attend_ref, _attention, _check_attend, _kind, _means_ref, _rand, _refusal, _rotary_ref, _rows, _run_attention, _t, _u, _view, gpu  # noqa: F401


# ------------------------------------------------------------------------------------------------ block selection

def _select_ref(q, mean, count, q_off, k_off, block, kv_heads, n_sel):
    """As the definition says, for many rows at once (numpy, 64 bits).  Equal means get one product, so that they tie."""
    group = q.shape[1] // kv_heads
    out = np.full((q.shape[0], kv_heads, n_sel), -7, np.int32)
    first = 0
    for a, b, ka, kb in zip(q_off, q_off[1:], k_off, k_off[1:]):
        nb = (kb - ka + block - 1) // block
        dead = count[first:first + nb] <= 0
        for g in range(kv_heads):
            of = np.ascontiguousarray(mean[first:first + nb, g])
            _, at, inverse = np.unique(of.view(np.dtype((np.void, of.shape[1] * 4))).reshape(-1), return_index=True, return_inverse=True)
            with np.errstate(all="ignore"):
                sc = (q[a:b, g * group:(g + 1) * group].astype(np.float64).sum(1) @ of[at].astype(np.float64).T)[:, inverse.reshape(-1)]
            nan = np.isnan(sc)
            if nan.any() or np.isinf(sc).any():
                order = np.lexsort((np.where(nan, 0.0, -sc), nan, np.broadcast_to(dead, sc.shape)))   # (stable: the lower block first)
            else:
                order = np.argsort(np.where(dead, np.inf, -sc), axis=1, kind="stable")
            n = min(n_sel, int((~dead).sum()))
            out[a:b, g] = -1
            out[a:b, g, :n] = np.sort(order[:, :n], axis=1)
        first += nb
    return out


def _select(gpu, dtype, q, mean, count, q_off, k_off, block, n_sel):
    pkg, ctx, torch = gpu
    md, cd = mean.cuda(), count.cuda()
    sel = torch.full((q.shape[0], mean.shape[1], n_sel), -7, dtype=torch.int32, device="cuda")
    ctx.block_select(pkg.block_select_args(pkg.offsets(q_off), pkg.offsets(k_off), dtype=_kind(pkg, dtype), head_dim=q.shape[2], block=block, q=_view(pkg, q),
                                           kv_heads=mean.shape[1], mean=md.data_ptr(), count=cd.data_ptr(), n_sel=n_sel, sel=sel.data_ptr()), pkg.STREAM_DEFAULT)
    return sel.cpu().numpy()


# rows of one set: 16 rows a work-group, and 32
FEW, MANY = [0, 300], [0, 2100]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, what, size", [(d, w, s) for w in ("query", "mean", "both") for s in (1e-20, 1e-25, 1e-37) for d in TYPES
                                               if d != "fp16" or w == "mean"])   # (fp16 holds no such query)
@pytest.mark.parametrize("q_off", (FEW, MANY), ids=("r300", "r2100"))
def test_block_select_of_very_short_vectors(gpu, dtype, what, size, q_off):
    """Queries or means (one of them in a hundred an exact zero) whose squares vanish in 32 bits, over means 1e-4 apart: the products
    are defined in 64 bits, whatever the vectors' length."""
    pkg, ctx, torch = gpu
    q = _rand(torch, 201, q_off[-1], 4, 64)
    mean = _rand(torch, 202, 1, 4, 64) + 1e-4 * _rand(torch, 203, 313, 4, 64)
    if what != "mean":
        q *= size
    if what != "query":
        mean *= size
    q[::100] = 0
    mean[7::100] = 0
    q = q.to(_t(torch, dtype))
    count = torch.full((313,), 32, dtype=torch.int32)
    got = _select(gpu, dtype, q.cuda(), mean, count, q_off, [0, 313 * 32], 32, 16)
    want = _select_ref(q.float().numpy(), mean.numpy(), count.numpy(), q_off, [0, 313 * 32], 32, 4, 16)
    assert np.array_equal(got, want), int((got != want).any(-1).sum())


# ------------------------------------------------------------------------------------------------ products far from zero

def _far_ref(torch, q, k, v, scale):
    """One key head, every query head against all of k, v [n][64]: (out, lse, tolerance without the type's roundings, sum p|v|).
    The products of these inputs are exact in 32 bits.  A weight's argument, its distance to a maximum that may be 8 binary orders
    (5.6) off, is off by 2^-21 of itself and the exponential by 2^-22; a sum as in test_attention.py; twice, for the numerator and the
    denominator."""
    z = (q.double() @ k.double().t()) * scale
    far = z - z.amax(-1, keepdim=True)
    p = torch.exp(far)
    total = p.sum(-1, keepdim=True)
    w = p / total
    t = w * (2.0 ** -20 * (7 + far.abs().clamp(max=1e4)) + 2 * (k.shape[0] / 32 + 64) * 2.0 ** -24)
    out, a = w @ v.double(), w @ v.double().abs()
    return out, (z.amax(-1, keepdim=True) + torch.log(total))[..., 0], t @ v.double().abs() + t.sum(-1, keepdim=True) * a, a


# name -> (A, B, scale): products are +-A^2 + B x, x = 0..7
FAR = {"2^28": (2.0 ** 14, 32.0, 0.11), "2^40": (2.0 ** 20, 2.0 ** 17, 1.0), "3e38": (5.5, 2.0 ** -3, 1e37), "6e38": (8.0, 2.0 ** -3, 1e37)}
# form -> (queries, heads, kv_heads, keys, places of a list): what the rules in attn_mfma.hip make of them
FAR_FORMS = {"rows": (3, 2, 2, 300, 0), "rows, shared keys": (2, 1, 1, 40000, 0), "tiles": (8300, 8, 1, 300, 0), "tiles, shared keys": (300, 4, 4, 9001, 0),
             "list": (3, 2, 2, 900, 6), "lists turned round": (700, 4, 4, 1500, 9)}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("form", FAR_FORMS)
def test_attention_products_far_from_zero(gpu, dtype, far, form):
    """scale * q.k of 2^24 to 2^40 and beyond what 32 bits hold, positive, negative and (the third of the query rows) near zero in
    one call: softmax depends on differences, so no row is empty or NaN.  The maximum climbs along the keys."""
    pkg, ctx, torch = gpu
    A, B, scale = FAR[far]
    if dtype == "fp16" and A > 65504:
        pytest.skip("fp16 holds no such query")
    nq, heads, kvh, n, places = FAR_FORMS[form]
    t = _t(torch, dtype)
    q, k = torch.zeros(nq, heads, 64), torch.zeros(n, kvh, 64)
    q[0::3, :, 0], q[1::3, :, 0], q[2::3, :, 0] = A, -A, 0
    q[:, :, 1] = B
    k[:, :, 0] = A
    k[:, :, 1] = (torch.arange(n) * 8 // n)[:, None].float()
    k[:, :, 1] += ((torch.arange(n) * 7919 % 11) == 0)[:, None].float() * -1      # (some keys fall back by one)
    v = _rand(torch, 211, n, kvh, 64).to(t)
    q, k = q.to(t), k.to(t)
    sel = None
    keys = torch.arange(n)
    if places:
        blocks = (n + 63) // 64
        sel = torch.arange(places, dtype=torch.int32)[None, None].repeat(nq, kvh, 1) * 2 % blocks
        keys = torch.cat([torch.arange(i * 64, min(n, i * 64 + 64)) for i in sel[0, 0].tolist()])
    for with_lse in (True, False):
        out, lse = _run_attention(gpu, dtype, q.cuda(), k.cuda(), v.cuda(), scale, [0, nq], [0, n], sel=None if sel is None else sel.cuda(), block=64 if places else 0,
                                  lse=with_lse)
        for h in range(heads):
            g = h // (heads // kvh)
            ref, rl, tol, a = _far_ref(torch, q[:3, h], k[keys, g], v[keys, g], scale)
            tol = tol + (0 if dtype == "fp32" else _u(dtype) * a * 1.01) + _u(dtype) * ref.abs() * 1.01
            if dtype == "fp16":
                tol = tol + 2.0 ** -25 * (v[keys, g].double().abs().sum(0) + 1)
            got = out[:, h].cpu().double()
            for r in range(3):
                err = (got[r::3] - ref[min(r, nq - 1)]).abs()
                assert (err <= tol[min(r, nq - 1)]).all(), (r, h, float(err.max()), got[r, :4].tolist() if r < nq else None)
            if with_lse:
                got_l = lse[:, h].cpu().double()
                for r in range(min(3, nq)):
                    want = float(rl[r])
                    with np.errstate(over="ignore"):
                        beyond = np.isinf(np.float32(want))
                    assert ((got_l[r::3] == math.copysign(math.inf, want)) if beyond else ((got_l[r::3] - want).abs() <= 2.0 ** -21 * (abs(want) + 1))).all(), (r, h, want, got_l[r::3][:3])


# ------------------------------------------------------------------------------------------------ sums that cancel

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", (5, 900))
def test_selected_blocks_whose_values_cancel(gpu, dtype, queries):
    """Sums are held in 32 bits until the result is rounded, between the kernels too: with equal weights (a zero query) and blocks
    whose values nearly cancel, what is left is right.  A weight of 1 is exact in every type, so the result is off by the 32-bit sums
    ((keys / 32 + 64) 2^-24 of sum p|v|, for the numerator and the denominator) and one rounding."""
    pkg, ctx, torch = gpu
    t = _t(torch, dtype)
    q, k = torch.zeros(queries, 4, 64, dtype=t), _rand(torch, 221, 640, 4, 64).to(t)
    v = torch.full((640, 4, 64), 1000.0)
    v[64:128] = -1000
    v[320:384] = -1000
    v[torch.arange(640) % 64 == 5] += torch.where(v[torch.arange(640) % 64 == 5] > 0, 4.0, 8.0)
    v = v.to(t)
    sel = torch.tensor([0, 1, 4, 5], dtype=torch.int32)[None, None].repeat(queries, 4, 1)
    out, _ = _run_attention(gpu, dtype, q.cuda(), k.cuda(), v.cuda(), 0.125, [0, queries], [0, 640], sel=sel.cuda(), block=64)
    keys = torch.cat([torch.arange(64 * i, 64 * i + 64) for i in (0, 1, 4, 5)])
    want, a = v[keys].double().mean(0)[:1], v[keys].double().abs().mean(0)[:1]
    tol = 2 * (256 / 32 + 64) * 2.0 ** -24 * a + _u(dtype) * want.abs() * 1.01
    assert float(want.abs().min()) > 4 * float(tol.max())
    err = (out.cpu().double() - want[:, :1]).abs()
    assert (err <= tol[:, :1]).all(), (float(err.max()), float(tol.max()))


# ------------------------------------------------------------------------------------------------ the Python argument helpers

def test_offsets_that_do_not_belong_together_are_refused(pkg):
    """The entry points read n_sets + 1 of both lists: two of different lengths must not reach them."""
    for a, b in (([0, 5], [0, 7, 9]), ([0, 5, 6], [0, 7])):
        with pytest.raises(ValueError, match="sets"):
            _attention(pkg, q_off=pkg.offsets(a), k_off=pkg.offsets(b))
        with pytest.raises(ValueError, match="sets"):
            pkg.block_select_args(pkg.offsets(a), pkg.offsets(b), dtype=pkg.F32, head_dim=64, block=64, q=_rows(pkg), kv_heads=2, n_sel=4)


@pytest.mark.parametrize("values", ([0, 1 << 31], np.array([0, (1 << 32) + 5]), [0, 2.5], np.array([0.0, 3.0]), [], [[0, 5]]), ids=str)
def test_offsets_that_32_bits_do_not_hold_are_refused(pkg, values):
    with pytest.raises(ValueError, match="offsets"):
        pkg.offsets(values)


@pytest.mark.parametrize("kind", (np.int64, np.int16, np.uint32))
def test_offsets_of_other_types_mean_the_same(pkg, kind):
    """Straight into the helpers, without offsets(): not read as if they were 32-bit numbers."""
    a = _attention(pkg, q_off=np.array([0, 5], kind), k_off=np.array([0, 7], kind))
    assert _refusal(pkg, "ppg_attention", a)[1] == "ppg_attention: ctx is NULL" and a.n_sets == 1
    a = _attention(pkg, q_off=np.array([0, 5, 3], kind), k_off=np.array([0, 7, 9, 0][:3], kind))
    assert "q_off[2] = 3" in _refusal(pkg, "ppg_attention", a)[1]
    a = _attention(pkg, q_off=np.array([0, 99, 5, 99], kind)[::2], k_off=[0, 7])      # every second number of an array
    assert _refusal(pkg, "ppg_attention", a)[1] == "ppg_attention: ctx is NULL"


# ------------------------------------------------------------------------------------------------ forms of block selection

# (dim, heads, kv_heads, n_sel, rows of the sets, blocks of the sets).  The first five give 256 work-groups of 32 rows: registers for 320 blocks and
# for 1088, one stretch and several, ragged last work-groups; then the shapes of 16 rows
SELECT_FORMS = [
    (64, 8, 4, 16, [300, 257, 289, 320, 1, 31, 350, 333, 0, 290], [300, 17, 320, 1, 319, 64, 0, 250, 5, 128]),
    (32, 4, 4, 7, [2081], [1000]), (128, 4, 4, 64, [1200, 901], [1088, 321]), (64, 8, 8, 33, [500, 560, 3], [1300, 700, 2300]), (32, 8, 8, 64, [1040], [320]),
    (64, 4, 4, 16, [10, 18], [157, 25]), (32, 4, 1, 1, [10, 18], [94, 25]), (128, 8, 2, 64, [10, 18], [282, 100]), (32, 2, 1, 64, [33, 1], [3750, 100]),
    (128, 2, 1, 5, [16, 17], [1088, 1089]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nan", (False, True))
@pytest.mark.parametrize("form", SELECT_FORMS, ids=lambda f: "d%d_h%d_%d_n%d_r%d_b%d" % (f[0], f[1], f[2], f[3], sum(f[4]), sum(f[5])))
def test_block_select_forms(gpu, dtype, nan, form):
    """Every set has blocks without keys, blocks with equal means (live and dead), a zero mean and a hundred means that are almost equal;
    zero queries and strided queries; once all finite, once with a NaN in a live block and infinities in a query."""
    pkg, ctx, torch = gpu
    dim, heads, kvh, n_sel, ql, nbs = form
    block = 32
    q_off = np.cumsum([2] + ql).tolist()
    k_off = np.cumsum([3] + [max(0, b * block - 5 * (b % 2)) for b in nbs]).tolist()
    q = _rand(torch, 231, q_off[-1] + 3, heads, 2 * dim)
    mean, count = _rand(torch, 232, sum(nbs), kvh, dim), torch.full((sum(nbs),), block, dtype=torch.int32)
    g = torch.Generator().manual_seed(17)
    first = 0
    for nb, a, b in zip(nbs, q_off, q_off[1:]):
        m, c = mean[first:first + nb], count[first:first + nb]
        if nb > 8:
            near = torch.randperm(nb, generator=g)[:100]
            m[near] = 1.5 * _rand(torch, 233 + nb, 1, kvh, dim) + 1e-5 * _rand(torch, 234 + nb, len(near), kvh, dim)
            same = torch.randperm(nb, generator=g)[:5]
            m[same[1:]] = m[same[0]].clone()
            c[torch.randperm(nb, generator=g)[:nb // 6]] = 0
            m[7] = 0
            q[a + (b - a) // 2:a + (b - a) // 2 + 1] = 0
            if nan:
                c[3] = block
                m[3, kvh - 1, dim - 1] = float("nan")
                if b - a > 4:
                    q[a + 2, 0, dim] = float("inf")
                    q[a + 4, heads - 1, dim + 1] = -float("inf")
        first += nb
    q = q.to(_t(torch, dtype))
    qd = q.cuda()[:, :, dim:]
    got = _select(gpu, dtype, qd, mean, count, q_off, k_off, block, n_sel)
    want = _select_ref(q[:, :, dim:].float().numpy(), mean.numpy(), count.numpy(), q_off, k_off, block, kvh, n_sel)
    assert np.array_equal(got, want), int((got != want).any(-1).sum())
    # heads outermost: the same choice
    assert np.array_equal(_select(gpu, dtype, qd.transpose(0, 1).contiguous().transpose(0, 1), mean, count, q_off, k_off, block, n_sel), want)


# ------------------------------------------------------------------------------------------------ forms of attention

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", (32, 64, 128))
def test_shared_tiles_with_strides(gpu, dtype, dim):
    """Enough rows for the kernel that shares tiles: slices of a packed projection, heads outermost, a head and a row seen many times
    (stride 0), an output that is a slice; masked keys, with and without lse."""
    pkg, ctx, torch = gpu
    t, n, heads = _t(torch, dtype), 40 * 129, 8
    off = list(range(0, n + 1, 129))
    packed = _rand(torch, 241, n, 3, heads, dim).to(t)
    skip = (torch.rand(n, generator=torch.Generator().manual_seed(4)) < 0.1).to(torch.uint8)
    scale = 1 / math.sqrt(dim)
    q, k, v = packed[:, 0], packed[:, 1], packed[:, 2]
    pd = packed.cuda()
    qd, kd, vd, sd = pd[:, 0], pd[:, 1], pd[:, 2], skip.cuda()
    ref = _attend_ref(torch, q, k, v, scale, off, off, skip)
    outs = []
    for with_lse in (True, False):
        home = torch.full((n, 2, heads, dim), 3.0, dtype=t, device="cuda")
        out, lse = _run_attention(gpu, dtype, qd, kd, vd, scale, off, off, sd, out=home[:, 1], lse=with_lse)
        _check_attend(torch, dtype, out, lse, ref)
        assert (home[:, 0] == 3).all()
        outs.append(out.contiguous())
        x, y, z = (u.transpose(0, 1).contiguous().transpose(0, 1) for u in (qd, kd, vd))
        turned = torch.empty(heads, n, dim, dtype=t, device="cuda").transpose(0, 1)
        _run_attention(gpu, dtype, x, y, z, scale, off, off, sd, out=turned, lse=with_lse)
        assert torch.equal(turned.contiguous(), outs[-1])
    # one key head seen as eight, one value row seen by all keys (what comes out is that row), one query row seen by all
    ref = _attend_ref(torch, q, k[:, :1].expand(n, heads, dim), v, scale, off, off, skip)
    out, lse = _run_attention(gpu, dtype, qd, kd[:, :1].expand(n, heads, dim), vd, scale, off, off, sd)
    _check_attend(torch, dtype, out, lse, ref)
    ref = _attend_ref(torch, q[:1].expand(n, heads, dim), k, v[:1].expand(n, heads, dim), scale, off, off, skip)
    for with_lse in (True, False):
        out, lse = _run_attention(gpu, dtype, qd[:1].expand(n, heads, dim), kd, vd[:1].expand(n, heads, dim), scale, off, off, sd, lse=with_lse)
        _check_attend(torch, dtype, out, lse, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("form", ("tiles", "tiles, shared keys", "lists turned round"))
def test_many_rows_with_extreme_products(gpu, dtype, dim, form):
    """Products that grow or fall along the keys (the running maximum moves in every tile), that are all far below zero, infinite or NaN,
    for rows of three kinds side by side, with and without lse."""
    pkg, ctx, torch = gpu
    t = _t(torch, dtype)
    nq, heads, kvh, n = dict([("tiles", (8300, 8, 1, 700)), ("tiles, shared keys", (300, 4, 4, 9001)), ("lists turned round", (1100, 4, 4, 700))])[form]
    sel = keys = None
    if form == "lists turned round":
        sel = torch.arange(11, dtype=torch.int32)[None, None].repeat(nq, kvh, 1)       # (all of the set's blocks)
    v = _rand(torch, 251, n, kvh, dim).to(t)
    k = torch.zeros(n, kvh, dim)
    k[:, :, 0] = (torch.arange(n) * 700 // n * 0.25 - 90)[:, None]       # up to +85
    for case in ("up", "down", "low", "inf", "nan"):
        kk = k.clone()
        q = torch.zeros(nq, heads, dim)
        q[0::3, :, 0], q[1::3, :, 0], q[2::3, :, 0] = 1, 0.5, -1
        if case == "down":
            kk = kk.flip(0)
        elif case == "low":
            kk[:, :, 0] = -30000.0
        elif case == "inf":
            kk[:, :, 0] = -math.inf      # rows of the third kind: +inf, so NaN
        elif case == "nan":
            q[7] = float("nan")
        a, b = q.to(t), kk.to(t)
        few = [0, 1, 2, 7]
        ref = _attend_ref(torch, a[few], b, v, 1.0, [0, 4], [0, n], None)
        if case == "inf":
            for x in ref[2:]:
                x.nan_to_num_(0, 0, 0)
            ref[0][0::3], ref[1][0::3], ref[0][1], ref[1][1] = 0, -math.inf, 0, -math.inf
            ref[0][2], ref[1][2] = math.nan, math.nan
            ref[0][3], ref[1][3] = 0, -math.inf      # (row 7 is of the second kind)
        kind = [0 if r % 3 == 0 else 1 if r % 3 == 1 else 2 for r in range(nq)]
        kind[7] = 3
        full = [x[kind] for x in ref]
        for with_lse in (True, False):
            out, lse = _run_attention(gpu, dtype, a.cuda(), b.cuda(), v.cuda(), 1.0, [0, nq], [0, n], sel=None if sel is None else sel.cuda(), block=64 if sel is not None else 0,
                                      lse=with_lse)
            _check_attend(torch, dtype, out, lse, full)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_turned_lists_with_strides(gpu, dtype):
    """Lists turned round over slices of packed projections, heads outermost, stride 0; the output a slice."""
    pkg, ctx, torch = gpu
    t, n, nq, block, n_sel = _t(torch, dtype), 3001, 400, 64, 12
    packed, pq = _rand(torch, 261, n, 3, 4, 64).to(t), _rand(torch, 262, nq, 2, 8, 64).to(t)
    off_q, off_k = [0, 150, nq], [0, 1900, n]
    g = torch.Generator().manual_seed(6)
    sel = torch.stack([torch.randperm(17, generator=g)[:n_sel] for _ in range(nq * 4)]).view(nq, 4, n_sel).to(torch.int32)
    skip = (torch.rand(n, generator=g) < 0.1).to(torch.uint8)
    kd, qd, sd = packed.cuda(), pq.cuda(), skip.cuda()
    k, v, q = packed[:, 1], packed[:, 2], pq[:, 1]
    ref = _attend_ref(torch, q, k, v, 0.125, off_q, off_k, skip, sel, block, n_sel)
    home = torch.full((nq, 2, 8, 64), 3.0, dtype=t, device="cuda")
    out, lse = _run_attention(gpu, dtype, qd[:, 1], kd[:, 1], kd[:, 2], 0.125, off_q, off_k, sd, sel.cuda(), block, out=home[:, 1])
    _check_attend(torch, dtype, out, lse, ref)
    assert (home[:, 0] == 3).all()
    x, y, z = (u.transpose(0, 1).contiguous().transpose(0, 1) for u in (qd[:, 1], kd[:, 1], kd[:, 2]))
    turned = torch.empty(8, nq, 64, dtype=t, device="cuda").transpose(0, 1)
    _run_attention(gpu, dtype, x, y, z, 0.125, off_q, off_k, sd, sel.cuda(), block, out=turned, lse=False)
    assert torch.equal(turned.contiguous(), out.contiguous())
    ref = _attend_ref(torch, q, k[:, :1].expand(n, 4, 64), v[:, 1:2].expand(n, 4, 64), 0.125, off_q, off_k, skip, sel, block, n_sel)
    out, lse = _run_attention(gpu, dtype, qd[:, 1], kd[:, 1, :1].expand(n, 4, 64), kd[:, 2, 1:2].expand(n, 4, 64), 0.125, off_q, off_k, sd, sel.cuda(), block)
    _check_attend(torch, dtype, out, lse, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ("bf16", "fp32"))
def test_many_rows_against_far_ones(gpu, dtype):
    """Keys, values and queries whose last rows lie 2^31 components and more behind the first, in the kernels for many rows."""
    pkg, ctx, torch = gpu
    t, n, stride = _t(torch, dtype), 140, 1 << 24
    flat = torch.empty(n * stride, dtype=t, device="cuda")
    assert flat.numel() > 1 << 31
    k, v = flat.as_strided((n, 2, 64), (stride, 128, 1)), flat.as_strided((n, 2, 64), (stride, 128, 1), 64)
    far_q, far_out = flat.as_strided((n, 4, 64), (stride, 64, 1), 1024), flat.as_strided((n, 4, 64), (stride, 64, 1), 2048)
    src_k, src_v, src_q = _rand(torch, 271, n, 2, 64).to(t), _rand(torch, 272, n, 2, 64).to(t), _rand(torch, 273, n, 4, 64).to(t)
    k.copy_(src_k)
    v.copy_(src_v)
    far_q.copy_(src_q)
    # shared tiles: 256 tiles of each key head
    q_off, k_off = list(range(0, 128 * 129 + 1, 129)), [0] + [12 + i for i in range(128)]
    q = _rand(torch, 274, q_off[-1], 4, 64).to(t)
    ref = _attend_ref(torch, q, src_k, src_v, 0.125, q_off, k_off, None)
    for with_lse in (True, False):
        out, lse = _run_attention(gpu, dtype, q.cuda(), k, v, 0.125, q_off, k_off, lse=with_lse)
        _check_attend(torch, dtype, out, lse, ref)
    # lists turned round, also with far queries and results
    q = _rand(torch, 275, 1500, 4, 64).to(t)
    g = torch.Generator().manual_seed(8)
    sel = torch.stack([torch.randperm(5, generator=g)[:4] for _ in range(3000)]).view(1500, 2, 4).to(torch.int32)
    ref = _attend_ref(torch, q, src_k, src_v, 0.125, [0, 1500], [0, n], None, sel, 32, 4)
    out, lse = _run_attention(gpu, dtype, q.cuda(), k, v, 0.125, [0, 1500], [0, n], sel=sel.cuda(), block=32)
    _check_attend(torch, dtype, out, lse, ref)
    ref = _attend_ref(torch, src_q, src_k, src_v, 0.125, [0, n], [0, n], None)
    out, lse = _run_attention(gpu, dtype, far_q, k, v, 0.125, [0, n], [0, n], out=far_out)
    _check_attend(torch, dtype, out, lse, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq, nk", ((2600, 1060000), (1100, 640000)))
def test_turned_lists_of_many_entries_over_many_blocks(gpu, dtype, nq, nk):
    """More entries than a work-group holds in registers together with more blocks than it counts at a time: 33125 blocks in four
    shares, and 20000 in one (fewer entries than blocks)."""
    pkg, ctx, torch = gpu
    t, block, n_sel = _t(torch, dtype), 32, 16
    nb = (nk + block - 1) // block
    assert nq * n_sel > 16384 and (nb > 4 * 8192) == (nq * n_sel >= nb)
    q, k, v = _rand(torch, 281, nq, 1, 32).to(t), _rand(torch, 282, nk, 1, 32).to(t), _rand(torch, 283, nk, 1, 32).to(t)
    g = torch.Generator().manual_seed(10)
    sel = torch.randint(0, nb, (nq, 1, n_sel), generator=g, dtype=torch.int32)
    sel[::3, 0, 0] = nb - 1
    sel[::4, 0, 5] = -1
    sel[::5, 0, 6] = nb
    sel[1::3, 0, 1] = torch.arange(len(sel[1::3]), dtype=torch.int32) % 40       # (crowds at the front)
    scale = 1 / math.sqrt(32)
    ref = _attend_ref(torch, q, k, v, scale, [0, nq], [0, nk], None, sel, block, n_sel)
    out, lse = _run_attention(gpu, dtype, q.cuda(), k.cuda(), v.cuda(), scale, [0, nq], [0, nk], sel=sel.cuda(), block=block)
    _check_attend(torch, dtype, out, lse, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("lists", (False, True))
def test_work_that_is_missing_or_small_is_refused_for_calls_that_need_some(gpu, lists):
    pkg, ctx, torch = gpu
    nq, nk = (600, 5000) if lists else (1, 200000)
    q, k = torch.zeros(nq, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(nk, 4, 64, dtype=torch.bfloat16, device="cuda")
    sel = torch.zeros(nq, 4, 16, dtype=torch.int32, device="cuda")
    args = pkg.attention_args(pkg.offsets([0, nq]), pkg.offsets([0, nk]), dtype=pkg.BF16, head_dim=64, scale=1.0, q=_view(pkg, q), k=_view(pkg, k), v=_view(pkg, k),
                              out=_view(pkg, q), **(dict(block=64, n_sel=16, sel=sel.data_ptr()) if lists else {}))
    need = ctx.attention_work(args)
    assert need > 0
    work = torch.empty(need + 512, dtype=torch.uint8, device="cuda")
    for p, n in ((None, need), (work.data_ptr(), need - 1), (work.data_ptr() + 16, need)):
        args.work, args.work_bytes = p, n
        with pytest.raises(pkg.PPGError, match="work must be"):
            ctx.attention(args, pkg.STREAM_DEFAULT)


# ------------------------------------------------------------------------------------------------ forms of rotary positions and block means

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout, dim, rot, heads", ((0, 64, 64, 3), (0, 128, 124, 1), (1, 64, 64, 3), (1, 128, 124, 1), (1, 64, 60, 5), (1, 32, 28, 2), (1, 128, 64, 2)))
def test_rotary_of_many_rows(gpu, dtype, layout, dim, rot, heads):
    """16384 rows and more take 16 rows a work-group; 16403 + 5 leave a short last one in both tensors."""
    pkg, ctx, torch = gpu
    t = _t(torch, dtype)
    n, axes = (16403, 5), 2
    freq = torch.from_numpy(np.tile(pkg.rotary_frequencies(rot // 4, 640.0), 2)).cuda()
    x = [_rand(torch, 291 + i, m, heads, dim).to(t).cuda() for i, m in enumerate(n)]
    pos = [(torch.rand(m, axes, generator=torch.Generator().manual_seed(i)) * 640).cuda() for i, m in enumerate(n)]
    y = [torch.full_like(u, 7.0) for u in x]
    args = dict(dtype=_kind(pkg, dtype), head_dim=dim, rot_dim=rot, layout=layout, n_axes=axes, freq=freq.data_ptr())
    ctx.rotary(pkg.rotary_args(n, [p.data_ptr() for p in pos], [_view(pkg, u) for u in x], [_view(pkg, u) for u in y], **args), pkg.STREAM_DEFAULT)
    for u, w, p in zip(x, y, pos):
        ref, size = _rotary_ref(torch, u.cpu(), p.cpu(), freq.cpu(), rot, layout, axes, 0)
        tol = _u(dtype) * ref.abs() * 1.01 + size * 2.0 ** -21 + (2.0 ** -25 if dtype == "fp16" else 0)
        assert ((w.cpu().double() - ref).abs() <= tol).all()
        assert torch.equal(w[..., rot:], u[..., rot:])
    z = [u.clone() for u in x]
    ctx.rotary(pkg.rotary_args(n, [p.data_ptr() for p in pos], [_view(pkg, u) for u in z], [_view(pkg, u) for u in z], **args), pkg.STREAM_DEFAULT)
    assert all(torch.equal(a, b) for a, b in zip(y, z))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, dim, heads", (("fp32", 128, 9), ("fp32", 64, 35), ("bf16", 128, 17), ("fp16", 32, 67), ("fp32", 128, 16)))
def test_block_means_of_wide_rows(gpu, dtype, dim, heads):
    """Rows of more than 256 chunks of 16 bytes: several rounds, the last one of another width."""
    pkg, ctx, torch = gpu
    block, off = 64, [1, 300, 300, 463]
    k = _rand(torch, 295, off[-1], heads, dim).to(_t(torch, dtype))
    skip = (torch.rand(off[-1], generator=torch.Generator().manual_seed(5)) < 0.2).to(torch.uint8)
    k[skip != 0] = float("nan")
    nb = sum((b - a + block - 1) // block for a, b in zip(off, off[1:]))
    mean, count = torch.full((nb, heads, dim), 9.0, device="cuda"), torch.empty(nb, dtype=torch.int32, device="cuda")
    kd, sd = k.cuda(), skip.cuda()
    ctx.block_means(pkg.block_means_args(pkg.offsets(off), dtype=_kind(pkg, dtype), head_dim=dim, block=block, k=_view(pkg, kd), skip=sd.data_ptr(),
                                         mean=mean.data_ptr(), count=count.data_ptr()), pkg.STREAM_DEFAULT)
    ref, cnt = _means_ref(torch, k, off, block, skip)
    assert count.tolist() == cnt and ((mean.cpu().double() - ref).abs() <= 2.0 ** -24 * ref.abs() + 2.0 ** -45).all()
