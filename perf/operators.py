"""The attention operators of the matching side as measurable cases: rotary positions, block means, block selection, attention
between descriptor sets (whole sets, or the key blocks that a query selected).

`own` chooses between the plain forms (elementary torch operations in 32 bits, 64 where the definition says so) and the
library's entry points.  A set is what one frame or one local map contributes: rows of `heads` vectors of `dim` components.
"""
import math

import torch

own = False

_TORCH = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_DEV = "cuda:0"
_ctx = None
_pkg = None


def _context():
    """The package and one matcher context, made once per process as a program would."""
    global _ctx, _pkg
    if _ctx is None:
        import __graft_entry__
        _pkg = __graft_entry__.load_pkg()
        _ctx = _pkg.Context(_pkg.default_config(640, 480), matcher_only=True)
    return _pkg, _ctx


def _stream(pkg):
    return torch.cuda.current_stream().cuda_stream or pkg.STREAM_DEFAULT


# ---------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one frame pair at the default key-point cap, as a tracker without batching calls it: latency
        dict(name="rotary one frame", op="rotary", dtype="fp32", sets=1, q=500, k=487, heads=4, kv_heads=4, dim=64, rot=64,
             layout="half", axes=2, spread=0.0),
        # 64 camera streams of ragged frames
        dict(name="rotary 64 streams", op="rotary", dtype="bf16", sets=64, q=1024, k=1024, heads=4, kv_heads=4, dim=64, rot=64,
             layout="interleaved", axes=2, spread=0.3),
        # cross attention of one frame pair
        dict(name="attend one pair", op="attend", dtype="fp32", sets=1, q=500, k=487, heads=4, kv_heads=4, dim=64, skip=0.0,
             spread=0.0, lse=False),
        # self attention within the frames of 64 camera streams
        dict(name="attend 64 streams", op="attend", dtype="bf16", sets=64, q=1024, k=1024, heads=4, kv_heads=4, dim=64, skip=0.03,
             spread=0.3, lse=False),
        # the largest point sets the matcher takes on one work-group (8192 rows a side), four of them
        dict(name="attend 8192 rows", op="attend", dtype="bf16", sets=4, q=8192, k=8191, heads=2, kv_heads=2, dim=128, skip=0.0,
             spread=0.0, lse=False),
        # one query (a single point, or a frame's pooled descriptor) against a whole map
        dict(name="attend one row", op="attend", dtype="bf16", sets=1, q=1, k=400003, heads=4, kv_heads=4, dim=64, skip=0.05,
             spread=0.0, lse=True),
        # the block means of a local map and of a large one, made once per map update
        dict(name="means local map", op="means", dtype="fp32", sets=1, k=20011, kv_heads=4, dim=64, block=64, skip=0.05, spread=0.0),
        dict(name="means large map", op="means", dtype="bf16", sets=1, k=1000003, kv_heads=4, dim=64, block=64, skip=0.05, spread=0.0),
        # which blocks of the map each key point of a frame attends to
        dict(name="select one frame", op="select", dtype="fp32", sets=1, q=500, k=20011, heads=4, kv_heads=4, dim=64, block=64,
             n_sel=16, skip=0.05, spread=0.0),
        dict(name="select 8 streams", op="select", dtype="bf16", sets=8, q=1024, k=65537, heads=4, kv_heads=4, dim=64, block=64,
             n_sel=16, skip=0.05, spread=0.0),
        # and the attention over them
        dict(name="blocks one frame", op="blocks", dtype="fp32", sets=1, q=500, k=20011, heads=4, kv_heads=4, dim=64, block=64,
             n_sel=16, skip=0.05, spread=0.0, lse=True),
        dict(name="blocks 8 streams", op="blocks", dtype="bf16", sets=8, q=1024, k=65537, heads=4, kv_heads=4, dim=64, block=64,
             n_sel=16, skip=0.05, spread=0.0, lse=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "attend", "attend", "means", "select", "blocks", "blocks"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    dim = rng.choice([32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    c = dict(op=op, dtype=dtype, dim=dim, kv_heads=kv_heads, spread=rng.choice([0.0, 0.3, 0.9]))
    width = heads * dim
    if op == "means":
        c.update(sets=rng.choice([1, 3, 16]), block=rng.choice([32, 64, 128]), skip=rng.choice([0.0, 0.05, 0.5]))
        c["k"] = _log_int(rng, 200, int(1000003 * 512 / (2 * kv_heads * dim * (2 if dtype == "fp32" else 1)) / c["sets"]))
        return c
    c["heads"] = heads
    if op == "rotary":
        c.update(sets=rng.choice([1, 2, 8, 64]), axes=rng.choice([1, 2]), layout=rng.choice(["half", "interleaved"]),
                 rot=rng.choice([dim, dim // 2, dim - 4]))
        most = int(64 * 1024 * 256 / width / c["sets"] / (2 if dtype == "fp32" else 1))
        c["q"], c["k"] = _log_int(rng, 1, most), _log_int(rng, 1, most)
        return c
    if op == "attend":
        # products of 32 bits run at a sixteenth of the 16-bit rate
        c.update(sets=rng.choice([1, 1, 2, 8, 40]), skip=rng.choice([0.0, 0.05, 0.5]), lse=rng.choice([False, True]))
        most = 4 * 8192 * 8191 * 256 / (16 if dtype == "fp32" else 1) / c["sets"] / width
        c["q"] = _log_int(rng, 1, int(min(8192, max(2, most / 64))))
        c["k"] = _log_int(rng, 1, int(max(2, min(most / c["q"], 400003 * 256 / (kv_heads * dim) / c["sets"] / (2 if dtype == "fp32" else 1)))))
        return c
    c.update(sets=rng.choice([1, 1, 2, 8]), block=rng.choice([32, 64, 128]), n_sel=rng.choice([1, 7, 16, 32]), skip=rng.choice([0.0, 0.05, 0.5]))
    most_k = int(8 * 65537 * 256 / (kv_heads * dim) / c["sets"] / (2 if dtype == "fp32" else 1))
    c["k"] = _log_int(rng, 300, min(131072, most_k))
    per_row = c["sets"] * width * (c["n_sel"] * c["block"] * (16 if dtype == "fp32" else 1) if op == "blocks" else c["k"] // c["block"])
    most_row = 8 * 256 * 1024 * (16 * 64 if op == "blocks" else 1024)
    c["q"] = _log_int(rng, 1, max(2, min(1024, most_row // per_row)))
    if op == "blocks":
        c["lse"] = rng.choice([False, True])
    return c


def _lengths(n, sets, spread):
    """Ragged lengths of `sets` sets, from n down to about (1 - spread) n; no seed enters, so that every seed is the same work."""
    return [max(1, int(n * (1.0 - spread * ((i * 0.6180339887) % 1.0)))) for i in range(sets)]


def _offsets(lengths):
    off = [0]
    for n in lengths:
        off.append(off[-1] + n)
    return off


def _blocks(lengths, block):
    return [(n + block - 1) // block for n in lengths]


def work(case):
    c = case
    e = 4 if c["dtype"] == "fp32" else 2
    ks = _lengths(c["k"], c["sets"], c["spread"])
    if c["op"] == "means":
        n, nb = sum(ks), sum(_blocks(ks, c["block"]))
        return {"bytes": n * c["kv_heads"] * c["dim"] * e + n + nb * (c["kv_heads"] * c["dim"] * 4 + 4), "flops": n * c["kv_heads"] * c["dim"]}
    qs = _lengths(c["q"], c["sets"], c["spread"])
    w, kw = c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
    if c["op"] == "rotary":
        return {"bytes": 2 * (sum(qs) * w + sum(ks) * kw) * e + 4 * c["axes"] * (sum(qs) + sum(ks)),
                "flops": 3 * (sum(qs) * c["heads"] + sum(ks) * c["kv_heads"]) * c["rot"]}
    if c["op"] == "select":
        nb = _blocks(ks, c["block"])
        return {"bytes": sum(qs) * w * e + sum(nb) * (kw * 4 + 4) + 4 * sum(qs) * c["kv_heads"] * c["n_sel"],
                "flops": sum(2 * q * b * w for q, b in zip(qs, nb))}
    io = 2 * sum(qs) * w * e + (4 * sum(qs) * c["heads"] if c["lse"] else 0)
    if c["op"] == "attend":
        return {"bytes": io + 2 * sum(ks) * kw * e + (sum(ks) if c["skip"] else 0), "flops": sum(4 * q * k * w for q, k in zip(qs, ks))}
    # a key enters the bytes once if the lists can name it at all
    reach = [min(k, q * c["n_sel"] * c["block"]) for q, k in zip(qs, ks)]
    return {"bytes": io + 2 * sum(reach) * kw * e + 4 * sum(qs) * c["kv_heads"] * c["n_sel"],
            "flops": sum(4 * q * min(k, c["n_sel"] * c["block"]) * w for q, k in zip(qs, ks))}


# -------------------------------------------------------------------------------------------------------------- inputs

def _inputs(case, seed):
    """Descriptors after a learned projection: keys scatter around a centre per neighbourhood of the map, a query resembles one
    key of its set more than the others; some points are culled (skip)."""
    c = case
    g = torch.Generator(device=_DEV)
    g.manual_seed(1000003 * seed + 17)
    t = _TORCH[c["dtype"]]
    ks = _lengths(c["k"], c["sets"], c["spread"])
    nk, kvh, d = sum(ks), c["kv_heads"], c["dim"]
    s = dict(case=c, k_off=_offsets(ks))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=_DEV)

    size = c.get("block", 64)
    centres = normal((nk + size - 1) // size, kvh, d)
    s["k"] = (0.7 * centres.repeat_interleave(size, 0)[:nk] + 0.7 * normal(nk, kvh, d)).to(t)
    if c["op"] != "means":
        qs = _lengths(c["q"], c["sets"], c["spread"])
        nq, h = sum(qs), c["heads"]
        s["q_off"] = _offsets(qs)
        lens = torch.tensor(ks, device=_DEV).repeat_interleave(torch.tensor(qs, device=_DEV))
        base = torch.tensor(s["k_off"][:-1], device=_DEV).repeat_interleave(torch.tensor(qs, device=_DEV))
        like = base + (torch.rand(nq, generator=g, device=_DEV) * lens).long().clamp_(max=max(ks) - 1).minimum(lens - 1)
        s["q"] = (0.8 * s["k"][like].float().repeat_interleave(h // kvh, 1) + 0.8 * normal(nq, h, d)).to(t)
    if c.get("skip"):
        s["skip"] = (torch.rand(nk, generator=g, device=_DEV) < c["skip"]).to(torch.uint8)
        s["skip"][torch.tensor(s["k_off"][:-1], device=_DEV)] = 0  # every set keeps a point
    else:
        s["skip"] = None
    if c["op"] == "rotary":
        # pixel coordinates on two axes, or one running index; frequencies fall from one radian per pixel to a turn per image
        rate = c["rot"] // 2 // c["axes"]
        j = torch.arange(rate, device=_DEV, dtype=torch.float64) / rate
        s["freq"] = (2 * math.pi / 1024) ** j.repeat(c["axes"]) if c["axes"] == 2 else 10000.0 ** -j
        if c["axes"] == 2 and c["rot"] % 4:
            raise ValueError("two axes need a multiple of four rotated components")
        for x, n in (("q", sum(qs)), ("k", nk)):
            s[x + "_pos"] = torch.rand(n, 2, generator=g, device=_DEV) * 1024 if c["axes"] == 2 else torch.arange(n, device=_DEV, dtype=torch.float32)[:, None] + 0.0
    if c["op"] in ("attend", "blocks"):
        s["v"] = normal(nk, kvh, d).to(t)
        s["scale"] = 1.0 / math.sqrt(d)
    if c["op"] in ("select", "blocks"):
        s["mean"], s["count"] = _plain_means(s)
    if c["op"] == "blocks":
        s["sel"] = _plain_select(s)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    pkg, ctx = _context()
    c = case
    kind = {"fp32": pkg.F32, "bf16": pkg.BF16, "fp16": pkg.F16}[c["dtype"]]

    def rows(x):
        return pkg.Rows(x.data_ptr(), x.shape[1], x.stride(0), x.stride(1))

    off = {x: pkg.offsets(s[x]) for x in ("q_off", "k_off") if x in s}
    skip = s["skip"].data_ptr() if s["skip"] is not None else None
    if c["op"] == "rotary":
        s["out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        s["args"] = pkg.rotary_args(dtype=kind, head_dim=c["dim"], rot_dim=c["rot"], n_axes=c["axes"], freq=s["freq"].data_ptr(),
                                    layout=pkg.ROTARY_HALF if c["layout"] == "half" else pkg.ROTARY_INTERLEAVED,
                                    n_rows=(len(s["q"]), len(s["k"])), pos=(s["q_pos"].data_ptr(), s["k_pos"].data_ptr()),
                                    src=(rows(s["q"]), rows(s["k"])), dst=(rows(s["out"][0]), rows(s["out"][1])))
    elif c["op"] == "means":
        nb = sum(_blocks(_lengths(c["k"], c["sets"], c["spread"]), c["block"]))
        s["out"] = torch.empty(nb, c["kv_heads"], c["dim"], device=_DEV), torch.empty(nb, dtype=torch.int32, device=_DEV)
        s["args"] = pkg.block_means_args(dtype=kind, head_dim=c["dim"], block=c["block"], k_off=off["k_off"], k=rows(s["k"]), skip=skip,
                                         mean=s["out"][0].data_ptr(), count=s["out"][1].data_ptr())
    elif c["op"] == "select":
        s["out"] = torch.empty(len(s["q"]), c["kv_heads"], c["n_sel"], dtype=torch.int32, device=_DEV)
        s["args"] = pkg.block_select_args(dtype=kind, head_dim=c["dim"], block=c["block"], q_off=off["q_off"], k_off=off["k_off"],
                                          q=rows(s["q"]), kv_heads=c["kv_heads"], mean=s["mean"].data_ptr(), count=s["count"].data_ptr(),
                                          n_sel=c["n_sel"], sel=s["out"].data_ptr())
    else:
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(s["q"].shape[:2], device=_DEV) if c["lse"] else None
        sparse = dict(block=c["block"], n_sel=c["n_sel"], sel=s["sel"].data_ptr()) if c["op"] == "blocks" else {}
        s["args"] = pkg.attention_args(dtype=kind, head_dim=c["dim"], scale=s["scale"], q_off=off["q_off"], k_off=off["k_off"],
                                       q=rows(s["q"]), k=rows(s["k"]), v=rows(s["v"]), out=rows(s["out"]), skip=skip,
                                       lse=s["lse"].data_ptr() if c["lse"] else None, **sparse)
        need = ctx.attention_work(s["args"])
        s["work"] = torch.empty(max(need, 1), dtype=torch.uint8, device=_DEV)
        s["args"].work, s["args"].work_bytes = s["work"].data_ptr(), need
    return s


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        stream = _stream(_pkg)
        if op == "rotary":
            _ctx.rotary(s["args"], stream)
        elif op == "means":
            _ctx.block_means(s["args"], stream)
        elif op == "select":
            _ctx.block_select(s["args"], stream)
        else:
            _ctx.attention(s["args"], stream)
            return (s["out"], s["lse"]) if s["lse"] is not None else s["out"]
        return s["out"]
    if op == "rotary":
        return _plain_rotary(s, "q"), _plain_rotary(s, "k")
    if op == "means":
        return _plain_means(s)
    if op == "select":
        return _plain_select(s)
    out, lse = _plain_attend(s) if op == "attend" else _plain_blocks(s)
    return (out, lse) if s["case"]["lse"] else out


# --------------------------------------------------------------------------------------------------------- plain forms

def _plain_rotary(s, which):
    c, x, pos = s["case"], s[which].float(), s[which + "_pos"].double()
    half = c["rot"] // 2
    axis = torch.arange(half, device=_DEV) // (half // c["axes"])
    a = pos[:, axis] * s["freq"]  # angles of far positions need 64 bits
    cos, sin = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    if c["layout"] == "half":
        u, v = x[..., :half], x[..., half:c["rot"]]
        y = torch.cat((u * cos - v * sin, u * sin + v * cos, x[..., c["rot"]:]), -1)
    else:
        u, v = x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2]
        y = torch.cat((torch.stack((u * cos - v * sin, u * sin + v * cos), -1).flatten(-2), x[..., c["rot"]:]), -1)
    return y.to(s[which].dtype)


def _plain_means(s):
    """Sums of a block in 64 bits: which block is chosen later must not hang on their order."""
    c, size = s["case"], s["case"]["block"]
    means, counts = [], []
    for a, b in zip(s["k_off"], s["k_off"][1:]):
        nb = (b - a + size - 1) // size
        keep = torch.ones(b - a, device=_DEV) if s["skip"] is None else (s["skip"][a:b] == 0).float()
        keep = torch.cat((keep, keep.new_zeros(nb * size - (b - a)))).view(nb, size)
        k = torch.cat((s["k"][a:b], s["k"].new_zeros(nb * size - (b - a), c["kv_heads"], c["dim"])))
        k = k.view(nb, size, c["kv_heads"], c["dim"])
        n = keep.sum(1)
        step = max(1, (1 << 27) // (size * c["kv_heads"] * c["dim"]))
        total = torch.cat([(k[i:i + step].double() * keep[i:i + step, :, None, None]).sum(1) for i in range(0, nb, step)])
        means.append((total / n.clamp(min=1).double()[:, None, None]).float())
        counts.append(n.to(torch.int32))
    return torch.cat(means), torch.cat(counts)


def _plain_select(s):
    """Scores of the summed heads of a group in 64 bits, ties to the lowest block; the chosen ones ascending, -1 behind them."""
    c, size, group = s["case"], s["case"]["block"], s["case"]["heads"] // s["case"]["kv_heads"]
    out, first = [], 0
    for (a, b), (ka, kb) in zip(zip(s["q_off"], s["q_off"][1:]), zip(s["k_off"], s["k_off"][1:])):
        nb = (kb - ka + size - 1) // size
        mean, live = s["mean"][first:first + nb].double(), s["count"][first:first + nb] > 0
        first += nb
        q = s["q"][a:b].double().view(b - a, c["kv_heads"], group, c["dim"]).sum(2)
        score = torch.matmul(q.transpose(0, 1).contiguous(), mean.permute(1, 2, 0).contiguous())
        score = score.masked_fill(~live, -math.inf)
        order = torch.sort(score, dim=-1, descending=True, stable=True)
        take = min(c["n_sel"], nb)
        idx = order.indices[..., :take].masked_fill(order.values[..., :take] == -math.inf, nb)
        idx = torch.sort(idx, dim=-1).values
        idx = idx.masked_fill(idx == nb, -1).to(torch.int32)
        idx = torch.cat((idx, idx.new_full((*idx.shape[:2], c["n_sel"] - take), -1)), -1)
        out.append(idx.transpose(0, 1))
    return torch.cat(out).contiguous()


def _softmax_times(score, v):
    """Rows of scores (-inf where masked) with their values: the weighted sum and the log of the sum of exponentials."""
    m = score.amax(-1, keepdim=True)
    safe = m.masked_fill(m == -math.inf, 0.0)
    p = torch.exp(score - safe)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / total.masked_fill(total == 0, 1.0)
    return o, (safe + torch.log(total))[..., 0]


def _plain_attend(s):
    c, group = s["case"], s["case"]["heads"] // s["case"]["kv_heads"]
    out = torch.empty(s["q"].shape, device=_DEV)
    lse = torch.empty(s["q"].shape[:2], device=_DEV)
    for (a, b), (ka, kb) in zip(zip(s["q_off"], s["q_off"][1:]), zip(s["k_off"], s["k_off"][1:])):
        step = max(1, (1 << 28) // ((kb - ka) * c["heads"]))
        kt = s["k"][ka:kb].float().permute(1, 2, 0).contiguous()
        v = s["v"][ka:kb].float().transpose(0, 1).contiguous()
        gone = None if s["skip"] is None else s["skip"][ka:kb] != 0
        for i in range(a, b, step):
            n = min(b, i + step) - i
            q = s["q"][i:i + n].float().view(n, c["kv_heads"], group, c["dim"]).permute(1, 2, 0, 3).reshape(c["kv_heads"], group * n, c["dim"])
            score = torch.matmul(q * s["scale"], kt)
            if gone is not None:
                score = score.masked_fill(gone, -math.inf)
            o, l = _softmax_times(score, v)
            out[i:i + n] = o.view(c["kv_heads"], group, n, c["dim"]).permute(2, 0, 1, 3).reshape(n, c["heads"], c["dim"])
            lse[i:i + n] = l.view(c["kv_heads"], group, n).permute(2, 0, 1).reshape(n, c["heads"])
    return out.to(s["q"].dtype), lse


def _plain_blocks(s):
    c, size, group = s["case"], s["case"]["block"], s["case"]["heads"] // s["case"]["kv_heads"]
    out = torch.empty(s["q"].shape, device=_DEV)
    lse = torch.empty(s["q"].shape[:2], device=_DEV)
    for (a, b), (ka, kb) in zip(zip(s["q_off"], s["q_off"][1:]), zip(s["k_off"], s["k_off"][1:])):
        step = max(1, (1 << 26) // (c["n_sel"] * size * c["dim"]))
        gone = torch.zeros(kb - ka, dtype=torch.bool, device=_DEV) if s["skip"] is None else s["skip"][ka:kb] != 0
        for h in range(c["kv_heads"]):
            k, v = s["k"][ka:kb, h].float(), s["v"][ka:kb, h].float()
            for i in range(a, b, step):
                n = min(b, i + step) - i
                idx = s["sel"][i:i + n, h].long()
                at = (idx[..., None] * size + torch.arange(size, device=_DEV)).view(n, -1)
                bad = (idx < 0).repeat_interleave(size, 1) | (at >= kb - ka)
                at = at.clamp(0, kb - ka - 1)
                bad = bad | gone[at]
                q = s["q"][i:i + n, h * group:(h + 1) * group].float() * s["scale"]
                score = torch.matmul(q, k[at].transpose(1, 2).contiguous()).masked_fill(bad[:, None], -math.inf)
                o, l = _softmax_times(score, v[at])
                out[i:i + n, h * group:(h + 1) * group] = o
                lse[i:i + n, h * group:(h + 1) * group] = l
    return out.to(s["q"].dtype), lse


# -------------------------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The definitions, set by set and head by head, in 64 bits."""
    s, c = _inputs(case, seed), case
    f64 = torch.float64
    if c["op"] == "rotary":
        res = []
        for x, pos in ((s["q"], s["q_pos"]), (s["k"], s["k_pos"])):
            y = x.to(f64).clone()
            half = c["rot"] // 2
            for j in range(half):
                i0, i1 = (j, j + half) if c["layout"] == "half" else (2 * j, 2 * j + 1)
                angle = pos[:, 0 if c["axes"] == 1 or j < half // 2 else 1].to(f64) * s["freq"][j]
                turn = torch.polar(torch.ones_like(angle), angle)[:, None] * torch.complex(x[..., i0].to(f64), x[..., i1].to(f64))
                y[..., i0], y[..., i1] = turn.real, turn.imag
            res.append(y)
        return tuple(res)
    sets = list(zip(s["k_off"], s["k_off"][1:]))
    if c["op"] == "means":
        nb = [(b - a + c["block"] - 1) // c["block"] for a, b in sets]
        total = torch.zeros(sum(nb), c["kv_heads"], c["dim"], dtype=f64, device=_DEV)
        count = torch.zeros(sum(nb), dtype=f64, device=_DEV)
        for (a, b), f in zip(sets, _offsets(nb)):
            at = f + torch.arange(b - a, device=_DEV) // c["block"]
            w = torch.ones(b - a, dtype=f64, device=_DEV) if s["skip"] is None else 1.0 - s["skip"][a:b].to(f64)
            for h in range(c["kv_heads"]):
                total[:, h].index_add_(0, at, s["k"][a:b, h].to(f64) * w[:, None])
            count.index_add_(0, at, w)
        return total / count.clamp(min=1.0)[:, None, None], count.to(torch.int32)
    if c["op"] == "select":
        # the chosen blocks are whole numbers that the plain form already computes in 64 bits
        return None
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=f64, device=_DEV)
    lse = torch.zeros(s["q"].shape[:2], dtype=f64, device=_DEV)
    for (a, b), (ka, kb) in zip(zip(s["q_off"], s["q_off"][1:]), sets):
        alive = torch.ones(kb - ka, dtype=torch.bool, device=_DEV) if s["skip"] is None else s["skip"][ka:kb] == 0
        for h in range(c["heads"]):
            g = h // group
            k, v = s["k"][ka:kb, g].to(f64), s["v"][ka:kb, g].to(f64)
            for i in range(a, b, 1024):
                n = min(b, i + 1024) - i
                z = s["q"][i:i + n, h].to(f64) @ k.t().contiguous() * s["scale"]
                allowed = alive.expand(n, kb - ka)
                if c["op"] == "blocks":
                    nb = (kb - ka + c["block"] - 1) // c["block"]
                    pick = torch.zeros(n, nb + 1, dtype=torch.bool, device=_DEV)
                    idx = s["sel"][i:i + n, g].long()
                    pick.scatter_(1, idx.masked_fill(idx < 0, nb), True)
                    allowed = allowed & pick[:, torch.arange(kb - ka, device=_DEV) // c["block"]]
                z = torch.where(allowed, z, torch.full_like(z, -math.inf))
                lse[i:i + n, h] = torch.logsumexp(z, 1)
                out[i:i + n, h] = torch.softmax(z, 1) @ v
    return (out, lse) if c["lse"] else out
