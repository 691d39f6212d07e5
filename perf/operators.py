"""What is measured of the state-space operators: the scan (prompts, packed prompts, training), the
single-token update and the slot maps that join them in serving.

Each case runs one operator once. With `own` false that is its plain form, elementary torch
operations in 32 bits rounded once at the end; with `own` true it is the call a user makes.

The recurrence, for each batch row, channel d and state n, with delta = softplus(dt + dt_bias):

    h[t] = exp(delta[t] A[d, n]) h[t-1] + delta[t] x[t] B[t, n]
    y[t] = sum_n C[t, n] h[t] + D[d] x[t],       out[t] = y[t] silu(z[t])
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"
_DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # One short prompt at the smallest configured width: launches and latency, not throughput.
        dict(name="prompt-short", op="scan", batch=1, seqlen=512, dim=512, state=16, groups=1, dtype="bfloat16", init=False),
        # A prompt chunk that continues from a kept state, at the streaming configuration's width.
        dict(name="prompt-chunk", op="scan", batch=2, seqlen=2048, dim=2048, state=16, groups=1, dtype="float16", init=True),
        # A batch of prompts at the streaming configuration's width.
        dict(name="prompt-batch", op="scan", batch=8, seqlen=2048, dim=2048, state=16, groups=1, dtype="bfloat16", init=False),
        # One long document: few rows, so the work has to be split along the sequence.
        dict(name="prompt-long", op="scan", batch=1, seqlen=32768, dim=1024, state=16, groups=1, dtype="bfloat16", init=False),
        # Serving: prompts of many requests packed in one row, each state left in its request's slot.
        dict(name="packed-prompts", op="packed", seqlen=8192, dim=2048, state=16, groups=1, dtype="bfloat16", requests=23),
        # A training step of a small model: the README's shape.
        dict(name="train-small", op="train", batch=2, seqlen=1024, dim=512, state=16, groups=1, dtype="bfloat16", init=False, packed=False),
        # A training step at the streaming configuration's width.
        dict(name="train-wide", op="train", batch=4, seqlen=2048, dim=2048, state=16, groups=1, dtype="bfloat16", init=False, packed=False),
        # Packed training rows in 32 bits with initial states; length, width, states all odd, B and C per group.
        dict(name="train-ragged-fp32", op="train", batch=3, seqlen=1021, dim=516, state=12, groups=3, dtype="float32", init=True, packed=True),
        # One new token of one request.
        dict(name="decode-one", op="update", batch=1, dim=512, state=16, groups=1, dtype="bfloat16", state_dtype="float32", slots=4),
        # One new token of a full batch of requests, states in slots.
        dict(name="decode-batch", op="update", batch=256, dim=4352, state=16, groups=1, dtype="bfloat16", state_dtype="float32", slots=288),
        # The maps of a small serving step.
        dict(name="maps-small", op="maps", requests=7, seqlen=512, width=4),
        # The maps of a large one.
        dict(name="maps-large", op="maps", requests=1024, seqlen=131072, width=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


#: A drawn scan or training case has at most this many (token, channel, state) triples: the largest listed one's.
_MOST_SCAN, _MOST_TRAIN = 32768 * 1024 * 16, 4 * 2048 * 2048 * 16


def draw(rng):
    op = rng.choice(["scan", "scan", "packed", "train", "train", "train", "update", "update", "maps"])
    if op == "maps":
        return dict(op=op, requests=_log(rng, 1, 1024), seqlen=_log(rng, 64, 131072), width=rng.randint(2, 8))
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    groups = rng.choice([1, 1, 1, 2, 4])
    state = rng.choice([16, 16, 16, 4, 8, 11, 32, 64])
    if op == "update":
        batch = _log(rng, 1, 256)
        return dict(op=op, batch=batch, dim=groups * _log(rng, 64 // groups, 4352 // groups), state=min(state, 16), groups=groups, dtype=dtype,
                    state_dtype=rng.choice(["float32", "float32", dtype]), slots=batch + rng.randint(0, 32))
    most = _MOST_TRAIN if op == "train" else _MOST_SCAN
    while True:
        batch = 1 if op == "packed" else _log(rng, 1, 16)
        seqlen = _log(rng, 1, 32768 if op == "scan" else 8192)
        dim = groups * _log(rng, max(1, 64 // groups), 4352 // groups)
        if rng.random() < 0.5:  # half of the widths are those of a model, half are any
            dim = max(64, dim // 64 * 64)
        if most / 4096 <= batch * seqlen * dim * state <= most and dim % groups == 0:
            break
    case = dict(op=op, batch=batch, seqlen=seqlen, dim=dim, state=state, groups=groups, dtype=dtype)
    if op == "packed":
        case.pop("batch")
        return dict(case, requests=rng.randint(1, max(1, min(64, seqlen // 8))))
    case["init"] = rng.random() < 0.5
    if op == "train":
        case["packed"] = rng.random() < 0.4
    return case


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _params(g, dim, state):
    """The decay rates, skip and step bias of a layer: A near -1..-N, steps between 1e-3 and 1e-1."""
    A = -torch.arange(1, state + 1, device=DEV, dtype=torch.float32) * torch.exp(0.1 * _randn(g, dim, state))
    step = torch.exp(_rand(g, dim) * (math.log(0.1) - math.log(1e-3)) + math.log(1e-3))
    return dict(A=A, D=1.0 + 0.1 * _randn(g, dim), dt_bias=step + torch.log(-torch.expm1(-step)))


def _tokens(g, case, batch, seqlen):
    """x after the convolution's SiLU, raw steps, gate, and B and C as the slices of one projection
    that a layer has them in (rows of 16 other columns, B, C)."""
    dt, dim, n, gr = _DT[case["dtype"]], case["dim"], case["state"], case["groups"]
    proj = _randn(g, batch, seqlen, 16 + 2 * gr * n).to(dt)
    B, C = proj[..., 16:16 + gr * n], proj[..., 16 + gr * n:]
    if gr > 1:
        B, C = B.unflatten(-1, (gr, n)), C.unflatten(-1, (gr, n))
    return dict(x=torch.nn.functional.silu(_randn(g, batch, seqlen, dim)).to(dt), dt=(0.5 * _randn(g, batch, seqlen, dim)).to(dt),
                z=_randn(g, batch, seqlen, dim).to(dt), B=B, C=C)


def _lengths(g, requests, seqlen):
    """Request lengths that fill about 15/16 of the row, one in eight of them zero where there are many."""
    share = -torch.log(_rand(g, requests).clamp_min(1e-6))
    if requests >= 8:
        share = share * (torch.arange(requests, device=DEV) % 8 != 5)
    fill = seqlen - seqlen // 16
    edges = torch.floor(torch.cumsum(share.double(), 0) / share.double().sum() * fill).long()
    return torch.diff(edges, prepend=edges.new_zeros(1)).to(torch.int32)


def _seq_idx(lengths, seqlen):
    edges = torch.cumsum(lengths.long(), 0)
    pos = torch.arange(seqlen, device=DEV)
    ids = torch.searchsorted(edges, pos, right=True)
    return torch.where(pos < edges[-1], ids, -1).to(torch.int32)[None]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    if op == "maps":
        r = case["requests"]
        lengths = _lengths(g, r, case["seqlen"])
        perm = torch.randperm(2 * r, generator=g, device=DEV).to(torch.int32)
        old = _rand(g, r) < 0.5  # half of the requests have a slot already
        return dict(case=case, lengths=lengths, slots=torch.where(old, perm[:r], -1).to(torch.int32), free=perm[r:].contiguous(),
                    past=torch.where(old, torch.randint(0, 4096, (r,), generator=g, device=DEV), 0).to(torch.int32))
    s = dict(case=case, **_params(g, case["dim"], case["state"]))
    dim, n = case["dim"], case["state"]
    if op == "update":
        b = case["batch"]
        s.update({k: v[:, 0] for k, v in _tokens(g, case, b, 1).items()})
        s["ssm_state"] = _randn(g, case["slots"], dim, n).to(_DT[case["state_dtype"]])
        s["slots"] = torch.randperm(case["slots"], generator=g, device=DEV)[:b].to(torch.int32)
        return s
    batch, seqlen = case.get("batch", 1), case["seqlen"]
    s.update(_tokens(g, case, batch, seqlen))
    s["init"] = _randn(g, batch, dim, n) if case.get("init") else None
    s["seq_idx"] = None
    if op == "packed":
        s["seq_idx"] = _seq_idx(_lengths(g, case["requests"], seqlen), seqlen)
        s["state_cache"] = _randn(g, case["requests"] + 3, dim, n)
        s["slots"] = torch.randperm(case["requests"] + 3, generator=g, device=DEV)[:case["requests"]].to(torch.int32)
    elif op == "train":
        if case["packed"]:
            s["seq_idx"] = torch.cat([_seq_idx(_lengths(g, max(1, min(9, seqlen // 4)), seqlen), seqlen) for _ in range(batch)])
        s["dout"] = _randn(g, batch, seqlen, dim).to(_DT[case["dtype"]])
        s["leaves"] = [k for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "init") if s[k] is not None]
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------
def _scan(a, b):
    """h[:, t] = a[:, t] h[:, t-1] + b[:, t] from h[:, -1] = 0: pairs of steps are joined to one of
    half the length, and the steps between follow from its result."""
    if a.shape[1] == 1:
        return b
    m = a.shape[1] // 2 * 2
    a1 = a[:, 1:m:2]
    odd = _scan(a1 * a[:, 0:m:2], a1 * b[:, 0:m:2] + b[:, 1:m:2])
    h = torch.empty_like(b)
    h[:, 0] = b[:, 0]
    h[:, 1::2] = odd
    h[:, 2::2] = a[:, 2::2] * odd[:, :(a.shape[1] - 1) // 2] + b[:, 2::2]
    return h


def _wide(v, dim):
    """(.., groups, n) or (.., n) of the groups to 32 bits at every channel: (.., dim, n) or (.., 1, n)."""
    v = v.float()
    return v[..., None, :] if v.ndim == 3 else v.repeat_interleave(dim // v.shape[2], 2)


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp_max(20))))


def _plain_forward(s):
    """What both directions need: the factors, the states and y before the gate."""
    x, dim = s["x"].float(), s["x"].shape[2]
    raw = s["dt"].float() + s["dt_bias"]
    delta, B, C, seq = _softplus(raw), _wide(s["B"], dim), _wide(s["C"], dim), s["seq_idx"]
    a = torch.exp(delta[..., None] * s["A"])
    b = (delta * x)[..., None] * B
    if seq is not None:
        cut = torch.zeros_like(seq, dtype=torch.bool)
        cut[:, 1:] = seq[:, 1:] != seq[:, :-1]
        off = seq < 0
        a = a * ~(cut | off)[..., None, None]
        b = b * ~off[..., None, None]
    if s["init"] is not None:
        b[:, 0] += a[:, 0] * s["init"]
    h = _scan(a, b)
    y = (h * C).sum(-1) + s["D"] * x
    if seq is not None:
        y = y * ~off[..., None]
    return x, raw, delta, B, C, a, h, y


def _plain_prompt(s):
    x, raw, delta, B, C, a, h, y = _plain_forward(s)
    z = s["z"].float()
    return (y * (z / (1 + torch.exp(-z)))).to(s["x"].dtype), h[:, -1].clone()


def _plain_packed(s):
    x, raw, delta, B, C, a, h, y = _plain_forward(s)
    z, seq = s["z"].float(), s["seq_idx"][0]
    last = (seq >= 0) & (torch.cat([seq[1:], seq.new_full((1,), -2)]) != seq)  # the last token of each request
    rows = last.nonzero()[:, 0]
    s["state_cache"][s["slots"][seq[rows]].long()] = h[0, rows]
    return (y * (z / (1 + torch.exp(-z)))).to(s["x"].dtype), s["state_cache"]


def _to_groups(v, like):
    """Sums a (batch, seqlen, dim, n) gradient over the channels that share a group."""
    if like.ndim == 3:
        return v.sum(2).to(like.dtype)
    return v.unflatten(2, (like.shape[2], -1)).sum(3).to(like.dtype)


def _plain_train(s):
    with torch.no_grad():
        x, raw, delta, B, C, a, h, y = _plain_forward(s)
        z, dout, dt_ = s["z"].float(), s["dout"].float(), s["x"].dtype
        sig = 1 / (1 + torch.exp(-z))
        dy = dout * z * sig
        dz = dout * y * sig * (1 + z * (1 - sig))
        if s["seq_idx"] is not None:
            dy = dy * (s["seq_idx"] >= 0)[..., None]
        # g[t] = dy[t] C[t] + a[t+1] g[t+1], the recurrence run backwards.
        nxt = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
        g = _scan(nxt.flip(1), (dy[..., None] * C).flip(1)).flip(1)
        prev = torch.zeros_like(h)
        prev[:, 1:] = h[:, :-1]
        if s["init"] is not None:
            prev[:, 0] = s["init"]
        q = g * prev * a  # the gradient of delta A
        gb = (g * B).sum(-1) if s["seq_idx"] is None else (g * B).sum(-1) * (s["seq_idx"] >= 0)[..., None]
        draw_ = ((q * s["A"]).sum(-1) + gb * x) / (1 + torch.exp(-raw))
        u = delta * x if s["seq_idx"] is None else delta * x * (s["seq_idx"] >= 0)[..., None]
        grads = dict(x=(delta * gb + s["D"] * dy).to(dt_), dt=draw_.to(dt_), A=(q * delta[..., None]).sum((0, 1)),
                     B=_to_groups(g * u[..., None], s["B"]), C=_to_groups(h * dy[..., None], s["C"]), D=(dy * x).sum((0, 1)),
                     z=dz.to(dt_), dt_bias=draw_.sum((0, 1)))
        if s["init"] is not None:
            grads["init"] = a[:, 0] * g[:, 0]
        return dict(out=(y * z * sig).to(dt_), **{"d" + k: v for k, v in grads.items()})


def _plain_update(s):
    x, dim, rows = s["x"].float(), s["x"].shape[1], s["slots"].long()
    delta = _softplus(s["dt"].float() + s["dt_bias"])
    B, C = (_wide(s[k][:, None], dim)[:, 0] for k in "BC")
    h = torch.exp(delta[..., None] * s["A"]) * s["ssm_state"][rows].float() + (delta * x)[..., None] * B
    z = s["z"].float()
    out = ((h * C).sum(-1) + s["D"] * x) * (z / (1 + torch.exp(-z)))
    s["ssm_state"][rows] = h.to(s["ssm_state"].dtype)
    return out.to(s["x"].dtype), s["ssm_state"]


def _plain_maps(s):
    """The edges of the requests in the packed row, each token's request and position, the rows that a
    convolution of `width` keeps of each request (-1 before its start), and the slots: a request with
    tokens and no slot takes the next free one."""
    n, seqlen, width = s["lengths"].long(), s["case"]["seqlen"], s["case"]["width"]
    edges = torch.cumsum(n, 0)
    cu = torch.cat([edges.new_zeros(1), edges])
    pos = torch.arange(seqlen, device=DEV)
    ids = torch.searchsorted(edges, pos, right=True)
    used = pos < edges[-1]
    at = ids.clamp_max(n.shape[0] - 1)
    seq_idx = torch.where(used, ids, -1)
    positions = torch.where(used, pos - cu[at] + s["past"][at], -1)
    tail = edges[:, None] - (width - 1) + torch.arange(width - 1, device=DEV)
    tail = torch.where(tail >= cu[:-1, None], tail, -1)
    new = (s["slots"] < 0) & (n > 0)
    rank = torch.cumsum(new, 0) - 1
    slots = torch.where(new, s["free"][rank.clamp_min(0)], s["slots"])
    i = torch.int32
    return cu.to(i), seq_idx[None].to(i), positions[None].to(i), tail.to(i), slots.to(i), new.sum().to(i)[None]


# ---------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------
def _api():
    path = os.path.join(os.getcwd(), "causal-conv1d-triton_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import causal_conv1d_b200

    return causal_conv1d_b200


def _own(s):
    api, op = _api(), s["case"]["op"]
    if op == "maps":
        return tuple(api.slot_maps_from_lengths(s["lengths"], s["case"]["seqlen"], width=s["case"]["width"], slots=s["slots"],
                                                free_slots=s["free"], past_lengths=s["past"]))
    args = (s["x"], s["dt"], s["A"], s["B"], s["C"])
    kw = dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"], dt_softplus=True)
    if op == "update":
        return api.ssm_update(s["x"], s["ssm_state"], *args[1:], ssm_state_indices=s["slots"], **kw), s["ssm_state"]
    if op == "packed":
        return api.ssm_scan(*args, seq_idx=s["seq_idx"], ssm_state=s["state_cache"], ssm_state_indices=s["slots"], **kw), s["state_cache"]
    if op == "scan":
        return api.ssm_scan(*args, initial_states=s["init"], return_final_states=True, **kw)
    out = api.ssm_scan(*args, seq_idx=s["seq_idx"], initial_states=s["init"], **kw)
    grads = torch.autograd.grad(out, [s[k] for k in s["leaves"]], s["dout"])
    return dict(out=out.detach(), **{"d" + k: v for k, v in zip(s["leaves"], grads)})


def run(s):
    if own:
        return _own(s)
    return {"scan": _plain_prompt, "packed": _plain_packed, "train": _plain_train, "update": _plain_update, "maps": _plain_maps}[s["case"]["op"]](s)


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "maps":
        r, t = case["requests"], case["seqlen"]
        return {"bytes": 4 * (2 * t + r * (5 + case["width"])), "flops": 0}
    es, dim, n, gr = torch.finfo(_DT[case["dtype"]]).bits // 8, case["dim"], case["state"], case["groups"]
    params = 4 * dim * (n + 2)
    if op == "update":
        tok, ss = case["batch"], torch.finfo(_DT[case["state_dtype"]]).bits // 8
        return {"bytes": tok * (es * (4 * dim + 2 * gr * n) + 2 * ss * dim * n) + params, "flops": tok * dim * (7 * n + 20)}
    batch = case.get("batch", 1)
    tok = batch * case["seqlen"]
    states = 4 * batch * dim * n
    if op == "train":  # x, dt, z, dout, B, C in; out, dx, ddt, dz, dB, dC out
        moved = tok * es * (8 * dim + 4 * gr * n) + 2 * params + (2 * states if case["init"] else 0) + (4 * tok if case["packed"] else 0)
        return {"bytes": moved, "flops": tok * dim * (24 * n + 60)}
    moved = tok * es * (4 * dim + 2 * gr * n) + params
    moved += (4 * tok + 4 * case["requests"] * dim * n) if op == "packed" else states * (2 if case["init"] else 1)
    return {"bytes": moved, "flops": tok * dim * (7 * n + 20)}


# ---------------------------------------------------------------------------------------------
# The same results from the definition, in 64 bits, one token after another
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "maps" or case.get("seqlen", 1) > 40000:
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_update(s) if case["op"] == "update" else _exact_sequence(s)


def _every_channel(v, dim):
    v = v.double()
    return v[:, None, :].expand(-1, dim, -1) if v.ndim == 2 else torch.repeat_interleave(v, dim // v.shape[1], dim=1)


def _exact_update(s):
    d = {k: s[k].double() for k in ("x", "dt", "A", "D", "z", "dt_bias")}
    step, rows, dim = torch.nn.functional.softplus(d["dt"] + d["dt_bias"]), s["slots"].long(), d["x"].shape[1]
    B, C = _every_channel(s["B"], dim), _every_channel(s["C"], dim)
    state = s["ssm_state"].double()
    h = state[rows] * torch.exp(torch.einsum("bd,dn->bdn", step, d["A"])) + torch.einsum("bd,bdn->bdn", step * d["x"], B)
    state[rows] = h
    return (torch.einsum("bdn,bdn->bd", h, C) + d["x"] * d["D"]) * torch.nn.functional.silu(d["z"]), state


def _exact_sequence(s):
    op = s["case"]["op"]
    d = {k: s[k].double() for k in ("x", "dt", "A", "D", "z", "dt_bias")}
    batch, seqlen, dim = d["x"].shape
    n = d["A"].shape[1]
    seq = s["seq_idx"]
    live = torch.ones(batch, seqlen, device=DEV, dtype=torch.bool) if seq is None else seq >= 0
    joined = torch.ones(batch, seqlen, device=DEV, dtype=torch.bool)
    if seq is not None:
        joined[:, 1:] = seq[:, 1:] == seq[:, :-1]
    joined = (joined & live).double()[..., None, None]
    step = torch.nn.functional.softplus(d["dt"] + d["dt_bias"])
    u = step * d["x"] * live[..., None]
    first = torch.zeros(batch, dim, n, device=DEV, dtype=torch.float64) if s["init"] is None else s["init"].double()
    keep = torch.empty(batch, seqlen, dim, n, device=DEV, dtype=torch.float64) if op == "train" else None
    cache = s["state_cache"].double() if op == "packed" else None
    ids = seq[0].tolist() if op == "packed" else None
    slots = s["slots"].tolist() if op == "packed" else None
    y = torch.empty(batch, seqlen, dim, device=DEV, dtype=torch.float64)

    def decay(t):
        return torch.exp(step[:, t, :, None] * d["A"]) * joined[:, t]

    h = first
    for t in range(seqlen):
        h = torch.addcmul(u[:, t, :, None] * _every_channel(s["B"][:, t], dim), decay(t), h)
        y[:, t] = (h * _every_channel(s["C"][:, t], dim)).sum(-1)
        if keep is not None:
            keep[:, t] = h
        if ids is not None and ids[t] >= 0 and (t + 1 == seqlen or ids[t + 1] != ids[t]):
            cache[slots[ids[t]]] = h[0]
    y = (y + d["D"] * d["x"]) * live[..., None]
    out = y * torch.nn.functional.silu(d["z"])
    if op == "packed":
        return out, cache
    if op == "scan":
        return out, h
    dout, sig = s["dout"].double(), torch.sigmoid(d["z"])
    dy = dout * d["z"] * sig * live[..., None]
    grads = {k: torch.zeros(v.shape, device=DEV, dtype=torch.float64) for k, v in s.items() if k in s["leaves"]}
    grads["z"] = dout * y * (sig + d["z"] * sig * (1 - sig))
    grads["D"] = (dy * d["x"]).sum((0, 1))
    dstep = torch.empty_like(step)
    carry = torch.zeros_like(first)

    def fold(v, like):
        return v.sum(1) if like.ndim == 3 else v.reshape(batch, like.shape[2], -1, n).sum(2)

    for t in range(seqlen - 1, -1, -1):
        gone = carry + dy[:, t, :, None] * _every_channel(s["C"][:, t], dim)
        before = decay(t) * (keep[:, t - 1] if t else first)
        grads["C"][:, t] = fold(keep[:, t] * dy[:, t, :, None], s["C"])
        grads["B"][:, t] = fold(gone * u[:, t, :, None], s["B"])
        along = (gone * _every_channel(s["B"][:, t], dim)).sum(-1) * live[:, t, None]
        rate = gone * before
        dstep[:, t] = along * d["x"][:, t] + (rate * d["A"]).sum(-1)
        grads["x"][:, t] = along * step[:, t] + d["D"] * dy[:, t]
        grads["A"] += (rate * step[:, t, :, None]).sum(0)
        carry = gone * decay(t)
    if "init" in grads:
        grads["init"] = carry
    grads["dt"] = dstep * torch.sigmoid(d["dt"] + d["dt_bias"])
    grads["dt_bias"] = grads["dt"].sum((0, 1))
    return dict(out=out, **{"d" + k: grads[k] for k in s["leaves"]})
