"""Attention between descriptor sets where the sizes, layouts and values of test_attention.py do not lead: vectors so short that
their squares vanish, products far from zero, sums that cancel, and the forms of the kernels that only large or strided calls take.

References are in 64 bits; tolerances are those of test_attention.py unless a test derives its own."""
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
