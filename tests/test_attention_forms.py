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
            rows, inverse = np.unique(mean[first:first + nb, g], axis=0, return_inverse=True)
            with np.errstate(all="ignore"):
                sc = (q[a:b, g * group:(g + 1) * group].astype(np.float64).sum(1) @ rows.astype(np.float64).T)[:, inverse.reshape(-1)]
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
