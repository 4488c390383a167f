"""Measured cases of the expert-block operators of facedetection_amd.ops.

A residual block whose inner products are split over experts, as it runs on the rows a detector holds (the
rois of a frame, the positions of a feature map): the norm before the block, the route of the rows to their
experts, the experts' matrix products over ragged groups of rows, the weighted sum of a row's expert outputs,
and the norm after the block with its gate and residual scale.

``run`` computes an operator in its plain form from elementary torch operations (``own`` false)
or with the calls a user makes (``own`` true).  ``exact`` is the definition in 64 bits.

Sizes: 10 rois of a frame at the default settings, 6 000 rois of the dense-crowd frame, 68 x 120 = 8 160
positions of the stride-16 map of a 1080p frame and 130 560 of a micro-batch of 16; widths 2048 (head
features), 1024 (feature map) and 512 (the RPN's hidden width); 8 to 64 experts.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------
# cases
def listed():
    return [
        # a frame's 10 rois enter a block: one launch of a few kilobytes, latency is all there is
        dict(name="norm_enter_rois", op="norm", rows=10, width=2048, x="f32", h="", kind="rms", gate="", act="", k=0, post=False, pre=True),
        # the positions of one 1080p frame leave a block and enter the next: float32 residual stream, bf16 branch,
        # one sigmoid gate row for the frame
        dict(name="norm_exit_map", op="norm", rows=8160, width=1024, x="f32", h="bf16", kind="layer", gate="group", act="sigmoid", k=0, post=True,
             pre=True),
        # the rois of a dense crowd leave an expert block: the weighted sum of two experts' rows inside the norm
        dict(name="norm_exit_experts", op="norm", rows=6000, width=2048, x="bf16", h="bf16", kind="rms", gate="row", act="", k=2, post=True, pre=True),
        # one frame's rois choose their experts: latency
        dict(name="route_rois", op="route", rows=10, experts=8, k=2, x="f32", normalize=True, masked=False),
        # the positions of a micro-batch of 16 frames, some of them padding
        dict(name="route_maps", op="route", rows=130560, experts=64, k=4, x="f32", normalize=False, masked=True),
        # one frame's rois through gated experts: every expert's weights for two or three rows each
        dict(name="linear_rois", op="linear", rows=10, k=2, experts=8, inner=2048, out=1024, x="bf16", act="silu", gated=True, bias=False, gather=True,
             skew=0.0, masked=False),
        # odd everything: 11 experts, 1001 inputs, 333 outputs, float16, some rows not routed
        dict(name="linear_odd", op="linear", rows=777, k=3, experts=11, inner=1001, out=333, x="f16", act="gelu", gated=False, bias=True, gather=True,
             skew=1.0, masked=True),
        # a dense crowd's rois, second product of the experts: rows already in expert order
        dict(name="linear_crowd", op="linear", rows=6000, k=2, experts=8, inner=2048, out=2048, x="bf16", act="", gated=False, bias=False, gather=False,
             skew=0.3, masked=False),
        # one frame's positions in the framework's own float32, one expert each, uneven shares
        dict(name="linear_map_f32", op="linear", rows=8160, k=1, experts=16, inner=1024, out=512, x="f32", act="relu", gated=False, bias=True, gather=True,
             skew=0.7, masked=False),
        # the positions of a micro-batch through gated experts: the largest product
        dict(name="linear_maps", op="linear", rows=130560, k=2, experts=64, inner=1024, out=1024, x="bf16", act="silu", gated=True, bias=False, gather=True,
             skew=0.3, masked=False),
        # one frame's rois gather their two expert rows: latency
        dict(name="combine_rois", op="combine", rows=10, k=2, width=2048, x="bf16", masked=False),
        # a micro-batch's positions gather theirs: memory
        dict(name="combine_maps", op="combine", rows=130560, k=2, width=1024, x="bf16", masked=True),
    ]


LIMIT_FLOPS = 2.0 * 130560 * 2 * 1024 * 2048
LIMIT_BYTES = 1.6e9


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _even(rng, n):
    """A size as drawn (mostly odd) or the next multiple of 64, half and half."""
    return n if rng.random() < 0.5 else -(-n // 64) * 64


def draw(rng):
    op = rng.choice(["norm", "route", "linear", "linear", "linear", "combine"])
    t = rng.choice(["f32", "bf16", "bf16", "f16"])
    while True:
        rows = _log(rng, 1, 130560)
        if op == "norm":
            h = rng.choice(["", t, t])
            c = dict(op=op, rows=rows, width=_even(rng, _log(rng, 33, 4096)), x=rng.choice([t, "f32"]) if h else t, h=h,
                     kind=rng.choice(["rms", "layer"]), gate=rng.choice(["", "row", "group", "full"]) if h else "",
                     act=rng.choice(["", "sigmoid", "tanh"]) if h else "", k=rng.choice([0, 0, 1, 2, 4]) if h else 0,
                     post=bool(h) and rng.random() < 0.8, pre=(not h) or rng.random() < 0.8)
        elif op == "route":
            e = _log(rng, 2, 256)
            c = dict(op=op, rows=rows, experts=e, k=min(e, rng.randint(1, 8)), x=t, normalize=rng.random() < 0.5, masked=rng.random() < 0.5)
        elif op == "linear":
            e = _log(rng, 1, 128)
            c = dict(op=op, rows=rows, k=min(e, rng.randint(1, 4)), experts=e, inner=_even(rng, _log(rng, 16, 4096)), out=_even(rng, _log(rng, 16, 2048)),
                     x=t, act=rng.choice(["", "relu", "silu", "gelu"]), gated=rng.random() < 0.4, bias=rng.random() < 0.5,
                     gather=rng.random() < 0.7, skew=rng.choice([0.0, 0.5, 1.0]), masked=rng.random() < 0.3)
        else:
            c = dict(op=op, rows=rows, k=rng.randint(1, 8), width=_even(rng, _log(rng, 33, 4096)), x=t, masked=rng.random() < 0.5)
        w = work(c)
        # the plain form holds float32 copies: the whole of a case stays within the largest listed one's
        scale = 4 if op != "route" else 8
        if w["flops"] <= LIMIT_FLOPS * (0.25 if t == "f32" else 1.0) and w["bytes"] * scale <= LIMIT_BYTES * 4:
            return c


def _active(case):
    """Expected number of experts that get a row."""
    p = [(i + 1.0) ** -case["skew"] for i in range(case["experts"])]
    s = sum(p)
    return sum(1.0 - (1.0 - min(1.0, q / s)) ** (case["rows"] * case["k"]) for q in p)


def work(case):
    T, k = case["rows"], case.get("k", 0)
    if case["op"] == "norm":
        D, sx, sh = case["width"], SIZE[case["x"]], SIZE[case["h"] or case["x"]]
        b = T * D * sx                                             # x
        b += 4 * D * (int(case["post"]) + int(case["pre"])) * (2 if case["kind"] == "layer" else 1)
        if case["h"]:
            b += T * D * sh * max(1, k) + T * k * 8 + T * D * sx   # h, its slots and weights, the new x
            b += {"": 0, "row": D * 4, "group": _groups(T) * D * sh, "full": T * D * sh}[case["gate"]]
        b += T * D * sh * int(case["pre"])
        return {"bytes": b, "flops": T * D * (8 + 2 * k)}
    if case["op"] == "route":
        E = case["experts"]
        return {"bytes": T * E * SIZE[case["x"]] + T * k * 16 + 4 * (E + 1) + (T if case["masked"] else 0), "flops": T * E * (2 + k)}
    if case["op"] == "linear":
        K, N, S, s = case["inner"], case["out"], T * k, SIZE[case["x"]]
        n = N * (2 if case["gated"] else 1)
        b = _active(case) * n * (K + int(case["bias"])) * s + (T if case["gather"] else S) * K * s + S * N * s + 4 * (case["experts"] + 1)
        return {"bytes": b + (4 * S if case["gather"] else 0), "flops": 2.0 * S * n * K}
    D, s = case["width"], SIZE[case["x"]]
    return {"bytes": T * k * D * s + T * D * s + T * k * 8, "flops": 2.0 * T * k * D}


def _groups(rows):
    """Rows are in frames; a gate row for each: 16, 4 or 1 frames, whichever divides the rows."""
    return next(g for g in (16, 4, 1) if rows % g == 0)


# ---------------------------------------------------------------------------------------------------------
# inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _choice(g, rows, experts, k, skew, masked):
    """Sorted slots of a routing with uneven shares: (experts int32 [rows, k], slots [rows, k], rows [rows*k], offsets [experts+1])."""
    share = -skew * torch.log(torch.arange(1, experts + 1, device="cuda", dtype=torch.float32))
    noise = -torch.log(-torch.log(torch.rand((rows, experts), generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)))
    chosen = (share + noise).topk(k, dim=1).indices
    if masked:
        chosen = chosen.masked_fill((torch.rand((rows, 1), generator=g, device="cuda") < 0.05), experts)
    flat = chosen.reshape(-1)
    by_expert, order = torch.sort(flat, stable=True)
    offsets = torch.searchsorted(by_expert, torch.arange(experts + 1, device="cuda")).to(torch.int32)
    slots = torch.empty_like(flat)
    slots[order] = torch.arange(flat.numel(), device="cuda")
    slots = slots.masked_fill(flat == experts, -1).reshape(rows, k).to(torch.int32)
    source = (order // k).masked_fill(by_expert == experts, -1).to(torch.int32)
    return slots, source, offsets


def prepare(case, seed):
    g = _gen(seed)
    T = case["rows"]
    st = dict(case=case)
    if case["op"] == "norm":
        D, k = case["width"], case["k"]
        tx, th = DTYPES[case["x"]], DTYPES[case["h"] or case["x"]]
        # a residual stream grows over the blocks and has a few large channels
        big = 1.0 + 20.0 * (torch.rand((D,), generator=g, device="cuda") < 0.01)
        st["x"] = (_randn(g, T, D) * 2.0 * big + 0.1).to(tx)
        for name in ("post", "pre"):
            if case[name]:
                st[name + "_weight"] = 1.0 + 0.2 * _randn(g, D)
                st[name + "_bias"] = 0.1 * _randn(g, D) if case["kind"] == "layer" else None
        if case["h"]:
            st["h"] = _randn(g, T * max(1, k), D).to(th)
            if k:
                st["slots"], _, _ = _choice(g, T, max(8, k), k, 0.3, True)
                st["weights"] = torch.softmax(_randn(g, T, k), dim=1)
            if case["gate"]:
                rows = {"row": 1, "group": _groups(T), "full": T}[case["gate"]]
                v = _randn(g, rows, D)
                st["gate"] = v.reshape(D) if case["gate"] == "row" else v.to(th)
            st["scale"] = 0.7071
        return st
    if case["op"] == "route":
        E = case["experts"]
        st["logits"] = (1.5 * _randn(g, T, E)).to(DTYPES[case["x"]])
        st["mask"] = torch.rand((T,), generator=g, device="cuda") >= 0.03 if case["masked"] else None
        return st
    if case["op"] == "linear":
        K, E, k, t = case["inner"], case["experts"], case["k"], DTYPES[case["x"]]
        n = case["out"] * (2 if case["gated"] else 1)
        _, source, st["offsets"] = _choice(g, T, E, k, case["skew"], case["masked"])
        st["rows"] = source if case["gather"] else None
        st["x"] = _randn(g, T if case["gather"] else T * k, K).to(t)
        st["weight"] = (_randn(g, E, n, K) / math.sqrt(K)).to(t)
        st["bias"] = (0.3 * _randn(g, E, n)).to(t) if case["bias"] else None
        st["bounds"] = st["offsets"].tolist()          # the plain form slices by host numbers
        return st
    st["slots"], _, _ = _choice(g, T, max(8, case["k"]), case["k"], 0.3, case["masked"])
    st["weights"] = torch.softmax(_randn(g, T, case["k"]), dim=1)
    st["y"] = _randn(g, T * case["k"], case["width"]).to(DTYPES[case["x"]])
    return st


# ---------------------------------------------------------------------------------------------------------
# one pass
def run(st):
    return (_own if own else _plain)(st)


def _own(st):
    from facedetection_amd import ops
    c = st["case"]
    if c["op"] == "norm":
        if not c["h"]:
            return ops.block_norm(st["x"], st["pre_weight"], st["pre_bias"], kind=c["kind"], eps=EPS)
        return ops.residual_norm(st["x"], st["h"], post_weight=st.get("post_weight"), post_bias=st.get("post_bias"), gate=st.get("gate"),
                                 gate_activation=c["act"] or None, scale=st["scale"], pre_weight=st.get("pre_weight"),
                                 pre_bias=st.get("pre_bias"), kind=c["kind"], eps=EPS, slots=st.get("slots"), weights=st.get("weights"))
    if c["op"] == "route":
        r = ops.expert_route(st["logits"], c["k"], mask=st["mask"], normalize=c["normalize"])
        return [r.weights, r.experts, r.slots, r.offsets, r.rows]
    if c["op"] == "linear":
        return ops.expert_linear(st["x"], st["weight"], st["offsets"], rows=st["rows"], bias=st["bias"], activation=c["act"] or None, gated=c["gated"])
    return ops.expert_combine(st["y"], st["slots"], st["weights"])


def _norm32(v, weight, bias, kind):
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + EPS) * weight
    return v if bias is None else v + bias


def _sum32(y, slots, weights):
    acc = torch.zeros((slots.shape[0], y.shape[1]), dtype=torch.float32, device=y.device)
    for j in range(slots.shape[1]):
        s = slots[:, j].long()
        w = weights[:, j].masked_fill(s < 0, 0.0)
        acc += w[:, None] * y[s.clamp(min=0)].float()
    return acc


def _act32(v, name):
    if name == "relu":
        return v.clamp(min=0)
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-v))
    if name == "tanh":
        return torch.tanh(v)
    return v


def _plain(st):
    c = st["case"]
    if c["op"] == "norm":
        x = st["x"].float()
        if not c["h"]:
            return _norm32(x, st["pre_weight"], st["pre_bias"], c["kind"]).to(st["x"].dtype)
        h = _sum32(st["h"], st["slots"], st["weights"]) if c["k"] else st["h"].float()
        if c["post"]:
            h = _norm32(h, st["post_weight"], st["post_bias"], c["kind"])
        if c["gate"]:
            gate = _act32(st["gate"].float(), c["act"])
            if c["gate"] == "group":
                gate = gate.repeat_interleave(c["rows"] // gate.shape[0], dim=0)
            h = h * gate
        x = x + st["scale"] * h
        if not c["pre"]:
            return x.to(st["x"].dtype)
        return x.to(st["x"].dtype), _norm32(x, st["pre_weight"], st["pre_bias"], c["kind"]).to(st["h"].dtype)
    if c["op"] == "route":
        E, k = c["experts"], c["k"]
        v = st["logits"].float()
        if st["mask"] is not None:
            v = v.masked_fill(~st["mask"][:, None], -math.inf)
        top, chosen = torch.sort(v, dim=1, descending=True, stable=True)       # ties: the lowest index first
        top, chosen = top[:, :k], chosen[:, :k]
        none = top == -math.inf
        e = torch.exp(top - top[:, :1].masked_fill(none[:, :1], 0.0))
        total = e.sum(dim=1, keepdim=True) if c["normalize"] else torch.exp(v - top[:, :1]).sum(dim=1, keepdim=True)
        weights = (e / total).masked_fill(none, 0.0)
        flat = chosen.masked_fill(none, E).reshape(-1)
        by_expert, order = torch.sort(flat, stable=True)
        offsets = torch.searchsorted(by_expert, torch.arange(E + 1, device=v.device)).to(torch.int32)
        slots = torch.empty_like(flat)
        slots[order] = torch.arange(flat.numel(), device=v.device)
        slots = slots.masked_fill(flat == E, -1).reshape(-1, k).to(torch.int32)
        rows = (order // k).masked_fill(by_expert == E, -1).to(torch.int32)
        return [weights, chosen.masked_fill(none, -1).to(torch.int32), slots, offsets, rows]
    if c["op"] == "linear":
        b, N = st["bounds"], c["out"]
        S = st["x"].shape[0] if st["rows"] is None else st["rows"].shape[0]
        y = torch.zeros((S, N), dtype=st["x"].dtype, device=st["x"].device)
        for e in range(c["experts"]):
            if b[e + 1] == b[e]:
                continue
            x = st["x"][b[e]:b[e + 1]] if st["rows"] is None else st["x"][st["rows"][b[e]:b[e + 1]].long()]
            v = torch.matmul(x.float(), st["weight"][e].float().t())
            if st["bias"] is not None:
                v = v + st["bias"][e].float()
            y[b[e]:b[e + 1]] = (_act32(v[:, :N], c["act"]) * v[:, N:] if c["gated"] else _act32(v, c["act"])).to(y.dtype)
        return y
    return _sum32(st["y"], st["slots"], st["weights"]).to(st["y"].dtype)


# ---------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "route": _exact_route, "linear": _exact_linear, "combine": _exact_combine}[case["op"]](case, st)


def _blocks(rows, width):
    step = max(1, (1 << 26) // max(1, width))
    return [(i, min(rows, i + step)) for i in range(0, rows, step)]


def _layer64(v, w, b, kind):
    mean = v.mean(1, keepdim=True) if kind == "layer" else 0.0
    square = torch.mean((v - mean) ** 2, 1, keepdim=True)
    out = (v - mean) / torch.sqrt(square + EPS) * w.double()
    return out if b is None else out + b.double()


def _exact_norm(case, st):
    T, D = st["x"].shape
    new, nxt = [], []
    for lo, hi in _blocks(T, D):
        x = st["x"][lo:hi].double()
        if case["h"]:
            if case["k"]:
                s = st["slots"][lo:hi].long()
                w = torch.where(s >= 0, st["weights"][lo:hi].double(), 0.0)
                h = sum(w[:, j:j + 1] * st["h"][s[:, j].clamp(min=0)].double() for j in range(case["k"]))
            else:
                h = st["h"][lo:hi].double()
            if case["post"]:
                h = _layer64(h, st["post_weight"], st["post_bias"], case["kind"])
            if case["gate"]:
                gate = st["gate"].double().reshape(-1, D)
                gate = {"": gate, "sigmoid": torch.sigmoid(gate), "tanh": torch.tanh(gate)}[case["act"]]
                h = h * gate[torch.arange(lo, hi, device=x.device) // (T // gate.shape[0])]
            x = x + st["scale"] * h
            new.append(x)
        if case["pre"]:
            nxt.append(_layer64(x, st["pre_weight"], st["pre_bias"], case["kind"]))
    out = [torch.cat(v) for v in (new, nxt) if v]
    return out[0] if len(out) == 1 else tuple(out)


def _exact_route(case, st):
    import numpy as np
    T, E, k = case["rows"], case["experts"], case["k"]
    v = st["logits"].double().cpu().numpy()
    live = np.ones(T, bool) if st["mask"] is None else st["mask"].cpu().numpy()
    chosen = np.argsort(-v, axis=1, kind="stable")[:, :k]
    e = np.exp(v - v.max(axis=1, keepdims=True))
    part = np.take_along_axis(e, chosen, 1)
    weights = part / (part if case["normalize"] else e).sum(axis=1, keepdims=True)
    weights[~live] = 0.0
    chosen[~live] = -1
    slots = np.full((T, k), -1, np.int32)
    rows = np.full((T * k,), -1, np.int32)
    offsets = np.zeros((E + 1,), np.int32)
    for expert in range(E):
        t, j = np.nonzero(chosen == expert)          # row-major: by token, then by rank
        at = offsets[expert]
        offsets[expert + 1] = at + len(t)
        slots[t, j] = at + np.arange(len(t))
        rows[at:at + len(t)] = t
    return [weights, chosen.astype(np.int32), slots, offsets, rows]


def _exact_linear(case, st):
    N, b = case["out"], st["bounds"]
    S = case["rows"] * case["k"]
    y = torch.zeros((S, N), dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(zip(b[:-1], b[1:])):
        if lo == hi:
            continue
        w = st["weight"][e].double().t().contiguous()
        for i, j in _blocks(hi - lo, max(w.shape)):
            x = (st["x"][lo + i:lo + j] if st["rows"] is None else st["x"][st["rows"][lo + i:lo + j].long()]).double()
            v = x @ w
            if st["bias"] is not None:
                v += st["bias"][e].double()
            a = v[:, :N]
            if case["act"]:
                a = {"relu": torch.relu, "silu": lambda u: u * torch.sigmoid(u), "gelu": torch.nn.functional.gelu}[case["act"]](a)
            y[lo + i:lo + j] = a * v[:, N:] if case["gated"] else a
    return y


def _exact_combine(case, st):
    out = []
    for lo, hi in _blocks(case["rows"], case["width"] * case["k"]):
        s = st["slots"][lo:hi].long()
        w = torch.where(s >= 0, st["weights"][lo:hi].double(), 0.0)
        out.append((w[:, :, None] * st["y"][s.clamp(min=0)].double()).sum(1))
    return torch.cat(out)
