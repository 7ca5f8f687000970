"""The operators of a state-space layer and of the 4-bit products around it, as cases that can be timed and compared: one
pass each through the public entry points (nextsycl_amd.attn.Ops), inputs resident on the GPU.

Five kinds of pass ("op"):
  prompt    a prompt's rows through the short causal convolution and the selective scan (ns_ssm_prompt): y, the state
            behind the last row and the ring of raw rows that the next pass's convolution starts from
  step      one token, or a few in a row, of each of several sequences (ns_ssm_step): y, the sequences' states, their rings
  gated     the group RMS norm behind the scan with its gate (ns_norm_gated)
  residual  a block's output into the residual stream, and the norm in front of the next block (ns_norm_residual)
  q4        rows times 4-bit weights with group scales (ns_q4_product)"""
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
TAPS, EPS = 4, 1e-5


def listed():
    return [
        # a whole prompt through one layer
        {"name": "ssm_prompt_8k", "op": "prompt", "io": "bf16", "rows": 8192, "past": 0, "heads": 128, "head": 64, "state": 128, "groups": 8},
        # a chunk in the middle of a longer prompt, float32 rows, half the heads (the layer's share of one card of two)
        {"name": "ssm_prompt_chunk", "op": "prompt", "io": "f32", "rows": 2051, "past": 4099, "heads": 64, "head": 64, "state": 128, "groups": 4},
        # a short follow-up question, heads that are no power of two wide
        {"name": "ssm_prompt_turn", "op": "prompt", "io": "f16", "rows": 85, "past": 20011, "heads": 128, "head": 80, "state": 128, "groups": 8},
        # a token of one chat
        {"name": "ssm_token", "op": "step", "io": "f32", "slots": 1, "each": 1, "idle": 0, "heads": 128, "head": 64, "state": 128, "groups": 8},
        # a token of each of many chats, a few of them idle
        {"name": "ssm_tokens_64", "op": "step", "io": "bf16", "slots": 64, "each": 1, "idle": 5, "heads": 128, "head": 64, "state": 128, "groups": 8},
        # a token and its three drafts of each of three chats
        {"name": "ssm_verify", "op": "step", "io": "f16", "slots": 3, "each": 4, "idle": 1, "heads": 128, "head": 80, "state": 128, "groups": 8},
        # the norm behind the scan: a token, a prompt
        {"name": "gated_token", "op": "gated", "io": "f32", "rows": 1, "width": 8192, "groups": 8, "order": 0},
        {"name": "gated_prompt", "op": "gated", "io": "bf16", "rows": 8192, "width": 8192, "groups": 8, "order": 0},
        # the residual stream between two blocks: a token, a ragged prompt with a norm on both sides and a gate
        {"name": "residual_token", "op": "residual", "io": "f16", "stream": "f32", "rows": 1, "width": 4096, "post": False, "gate": False},
        {"name": "residual_prompt", "op": "residual", "io": "bf16", "stream": "f32", "rows": 4001, "width": 5120, "post": True, "gate": True},
        # a token's in-projection, every block of 32 weights with a scale
        {"name": "q4_token", "op": "q4", "io": "f16", "rows": 1, "out": 18560, "in": 4096, "group": 32},
        # a verify pass's out-projection, float32 rows, a scale for 128 weights
        {"name": "q4_verify", "op": "q4", "io": "f32", "rows": 8, "out": 4096, "in": 8192, "group": 128},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (heads, features a head, state, groups) of hybrid models' layers and their shares of a card
LAYERS = [(128, 64, 128, 8), (128, 80, 128, 8), (64, 64, 128, 4), (32, 64, 128, 2), (16, 64, 128, 1), (80, 64, 64, 1), (24, 64, 128, 1), (64, 32, 256, 2),
          (32, 128, 128, 8), (18, 50, 100, 2), (7, 64, 16, 7)]


def draw(rng):
    op = rng.choice(["prompt", "prompt", "prompt", "step", "step", "gated", "residual", "q4", "q4"])
    io = rng.choice(["f32", "f16", "bf16"])
    if op in ("prompt", "step"):
        H, P, N, G = rng.choice(LAYERS)
    if op == "prompt":
        past = rng.choice([0, _log(rng, 1, 100000)])
        rows = _log(rng, 1, min(8192 if io != "f32" else 4096, 8192 * 128 * 64 // (H * P)))
        if past:
            rows = max(0, rows - 8) // 8 * 8 + rng.choice([3, 4, 5])        # (see _prepare_prompt)
        return {"op": op, "io": io, "rows": rows, "past": past, "heads": H, "head": P, "state": N, "groups": G}
    if op == "step":
        each = rng.choice([1, 1, rng.randint(2, 8)])
        return {"op": op, "io": io, "slots": max(1, _log(rng, 1, 64) // each), "each": each, "idle": rng.randint(0, 3), "heads": H, "head": P, "state": N, "groups": G}
    if op == "gated":
        groups = rng.choice([1, 2, 4, 8])
        width = groups * _log(rng, 16, 8192 // groups)
        return {"op": op, "io": io, "rows": min(_log(rng, 1, 8192), 8192 * 4096 // width), "width": width, "groups": groups, "order": rng.randint(0, 1)}
    if op == "residual":
        width = _log(rng, 32, 16384)
        return {"op": op, "io": io, "stream": rng.choice(["f32", io]), "rows": min(_log(rng, 1, 8192), 4001 * 5120 // width), "width": width,
                "post": rng.random() < 0.5, "gate": rng.random() < 0.5}
    return {"op": op, "io": io, "rows": rng.choice([1, 1, rng.randint(2, 16)]), "out": _log(rng, 64, 18560), "in": _log(rng, 64, 8192 if io != "f32" else 4096),
            "group": rng.choice([32, 64, 128])}


# ---- what a program has in hand before the call

class _Random:
    def __init__(self, seed):
        self.g = torch.Generator("cuda").manual_seed(seed)

    def __call__(self, *shape, sigma=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g, device="cuda") * sigma).to(dtype)

    def uniform(self, lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(*shape, generator=self.g, device="cuda")

    def whole(self, hi, *shape):
        return torch.randint(0, hi, shape, generator=self.g, device="cuda")


def prepare(case, seed):
    s = {"prompt": _prepare_prompt, "step": _prepare_step, "gated": _prepare_gated, "residual": _prepare_residual, "q4": _prepare_q4}[case["op"]](case, _Random(seed))
    s["case"] = case
    torch.cuda.synchronize()      # torch's stream and the library's are two
    return s


def _sizes(c):
    H, P, N, G = c["heads"], c["head"], c["state"], c["groups"]
    return H, P, N, G, H * P, H * P + 2 * G * N


def _layer(c, rand):
    """A layer's own weights: taps, bias, decay rates, the step size's bias, the skip."""
    H, P, N, G, inner, chan = _sizes(c)
    step = torch.exp(rand.uniform(math.log(1e-3), math.log(0.1), H))
    return {"cw": rand(chan, TAPS, sigma=0.5), "cb": rand(chan, sigma=0.1), "a": -rand.uniform(1.0, 16.0, H), "dtb": step + torch.log(-torch.expm1(-step)),
            "d": 1.0 + 0.1 * rand(H)}


def _prepare_prompt(c, rand):
    H, P, N, G, inner, chan = _sizes(c)
    T, p0, kind = c["rows"], c["past"], DTYPE[c["io"]]
    s = _layer(c, rand)
    # the in-projection's rows: gate | x B C | step sizes, one row
    s["row"] = inner + chan + H
    s["rows"] = rand(T, s["row"], dtype=kind)
    # the ring of raw rows, position % 8: where a pass continues a prompt, its length leaves the rows that it began from
    # beside those that it leaves behind, so that a pass can be timed again on the same state
    s["ring"] = rand(8, chan, dtype=kind).float()
    s["h0"] = rand(H, P, N, sigma=0.3) if p0 else None
    s["h1"] = torch.zeros(H, P, N, device="cuda")
    s["y"] = torch.zeros(T, inner, dtype=kind, device="cuda")
    return s


def _prepare_step(c, rand):
    H, P, N, G, inner, chan = _sizes(c)
    S, each, kind = c["slots"], c["each"], DTYPE[c["io"]]
    R, slots = S * each, S + c["idle"]
    s = _layer(c, rand)
    s["row"] = inner + chan + H
    s["rows"] = rand(R, s["row"], dtype=kind)
    # every sequence's rows follow each other; the sequences sit in slots of one allocation, in no order, some slots idle
    order = torch.argsort(rand(slots))[:S]
    s["slots"] = order.repeat_interleave(each).to(torch.int32)
    s["pos"] = rand.whole(100000, S).repeat_interleave(each).to(torch.int32) + torch.arange(each, device="cuda", dtype=torch.int32).repeat(S)
    s["cap"] = TAPS - 1 + each
    s["nslots"] = slots
    s["ring"] = rand(slots, s["cap"], chan, dtype=kind).float()
    s["h0"] = rand(slots, H, P, N, sigma=0.3)
    s["h1"] = torch.zeros(slots, H, P, N, device="cuda")
    s["y"] = torch.zeros(R, inner, dtype=kind, device="cuda")
    return s


def _prepare_gated(c, rand):
    T, D, kind = c["rows"], c["width"], DTYPE[c["io"]]
    return {"y": rand(T, D, dtype=kind), "z": rand(T, D, dtype=kind), "w": 1.0 + 0.1 * rand(D), "out": torch.empty(T, D, dtype=kind, device="cuda")}


def _prepare_residual(c, rand):
    T, D, kind, stream = c["rows"], c["width"], DTYPE[c["io"]], DTYPE[c["stream"]]
    s = {"x": rand(T, D, dtype=kind), "h": rand(T, D, sigma=3.0, dtype=stream), "pre": 1.0 + 0.1 * rand(D), "h1": torch.empty(T, D, dtype=stream, device="cuda"),
         "out": torch.empty(T, D, dtype=kind, device="cuda")}
    s["post"] = 1.0 + 0.1 * rand(D) if c["post"] else None
    s["gate"] = rand.uniform(0.2, 1.0, D) if c["gate"] else None
    s["scale"] = 0.22
    return s


def _q4_sizes(c):
    """Tiles of 16 outputs x 128 inputs: how many, and the scales' groups in each."""
    return (c["out"] + 15) // 16, (c["in"] + 127) // 128, 128 // c["group"]


def _prepare_q4(c, rand):
    T, M, K, kind = c["rows"], c["out"], c["in"], DTYPE[c["io"]]
    mt, kt, gr = _q4_sizes(c)
    # the weights as the engine holds them, tile by tile: 1024 bytes of nibbles (a lane's 16 bytes: output m of 16, and 8
    # inputs of each 32, input e in nibble e % 2 * 4 + e / 2), then the groups' half scales (4 outputs side by side)
    q = rand.whole(16, mt * 16, kt * 128)
    scale = (0.02 * torch.exp(0.3 * rand(mt * 16, kt * gr))).to(torch.float16)
    q[M:], q[:, K:], scale[M:] = 8, 8, 0
    scale[:, (K + c["group"] - 1) // c["group"]:] = 0
    n = q.view(mt, 16, kt, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 6, 5)             # tile, g, m, j, (e % 2, e / 2)
    n = n.reshape(mt, kt, 64, 4, 4, 2)                                          # (lane, j, byte, low / high)
    nib = (n[..., 0] | n[..., 1] << 4).to(torch.uint8).reshape(mt, kt, 1024)
    sc = scale.view(mt, 4, 4, kt, gr).permute(0, 3, 1, 4, 2).reshape(mt, kt, 16 * gr).contiguous().view(torch.uint8)
    return {"w": torch.cat([nib, sc.view(mt, kt, 32 * gr)], 2).contiguous(), "x": rand(T, K, dtype=kind), "y": torch.empty(T, M, dtype=kind, device="cuda")}


# ---- the plain forms

def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _softplus(v):
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-torch.abs(v)))


def _history(ring, p0):
    """The TAPS - 1 raw rows in front of position p0, the oldest first; zeros in front of the first."""
    at = torch.arange(p0 - TAPS + 1, p0, device=ring.device)
    return torch.where((at >= 0)[:, None], ring[at % ring.shape[0]], torch.zeros((), device=ring.device))


def _plain_prompt(c, s):
    H, P, N, G, inner, chan = _sizes(c)
    T, p0, L = c["rows"], c["past"], 64
    raw = s["rows"][:, inner:inner + chan].float()
    full = torch.cat([_history(s["ring"], p0), raw])
    u = _silu((torch.stack([full[k:k + T] for k in range(TAPS)]) * s["cw"].t()[:, None]).sum(0) + s["cb"])
    dt = _softplus(s["rows"][:, inner + chan:].float() + s["dtb"])
    # whole chunks: rows of zeros with a step of zero change nothing
    n = (T + L - 1) // L
    u = torch.cat([u, u.new_zeros(n * L - T, chan)])
    dt = torch.cat([dt, dt.new_zeros(n * L - T, H)])
    x = u[:, :inner].view(n, L, H, P).transpose(1, 2).contiguous()                                  # [n][H][L][P]
    B = u[:, inner:inner + G * N].view(n, L, G, N).transpose(1, 2).contiguous()                     # [n][G][L][N]
    C = u[:, inner + G * N:].view(n, L, G, N).transpose(1, 2).contiguous()
    dt = dt.view(n, L, H).transpose(1, 2).contiguous()                                              # [n][H][L]
    cum = torch.cumsum(dt.double() * s["a"].double()[:, None], 2)                                   # sums of a chunk's exponents, in 64 bits
    CB = torch.matmul(C, B.transpose(2, 3).contiguous())
    seen = torch.ones(L, L, dtype=torch.bool, device=u.device).tril()
    decay = torch.exp(torch.where(seen, cum[..., :, None] - cum[..., None, :], -math.inf).float())
    y = torch.matmul(CB.repeat_interleave(H // G, 1) * decay * dt[:, :, None, :], x)
    rest = (dt * torch.exp((cum[..., -1:] - cum).float()))[..., None]
    added = torch.matmul((x * rest).transpose(2, 3).contiguous(), B.repeat_interleave(H // G, 1))   # [n][H][P][N]
    # the state in front of each chunk, and behind the last: the chunks' own, each decayed by those between
    h0 = torch.zeros_like(s["h1"]) if s["h0"] is None else s["h0"]
    parts = torch.cat([h0[None], added]).transpose(0, 1).reshape(H, n + 1, P * N)
    ends = torch.cat([torch.zeros(1, H, dtype=torch.float64, device=u.device), torch.cumsum(cum[..., -1], 0)]).t()
    among = torch.ones(n + 1, n + 1, dtype=torch.bool, device=u.device).tril()
    between = torch.exp(torch.where(among, ends[:, :, None] - ends[:, None, :], -math.inf).float())
    states = torch.matmul(between, parts).view(H, n + 1, P, N)
    first = states[:, :n].permute(1, 0, 3, 2).contiguous()                                          # [n][H][N][P]
    y = y + torch.matmul(C.repeat_interleave(H // G, 1), first) * torch.exp(cum.float())[..., None] + x * s["d"][:, None, None]
    keep = torch.arange(max(0, T - TAPS + 1), T, device=u.device)
    s["ring"][(p0 + keep) % s["ring"].shape[0]] = raw[keep]
    return {"y": y.transpose(1, 2).reshape(n * L, inner)[:T].to(DTYPE[c["io"]]), "state": states[:, n].contiguous(), "ring": s["ring"]}


def _plain_step(c, s):
    H, P, N, G, inner, chan = _sizes(c)
    S, each = c["slots"], c["each"]
    slots = s["slots"].view(S, each)[:, 0].long()
    pos = s["pos"].view(S, each)[:, 0].long()
    rows = s["rows"].view(S, each, -1)
    raw = rows[..., inner:inner + chan].float()
    at = pos[:, None] + torch.arange(1 - TAPS, 0, device=pos.device)
    past = torch.where((at >= 0)[..., None], s["ring"][slots[:, None], at % s["cap"]], torch.zeros((), device=pos.device))
    full = torch.cat([past, raw], 1)
    dt = _softplus(rows[..., inner + chan:].float() + s["dtb"])
    h, out = s["h0"][slots], []
    for j in range(each):                                    # (a sequence's rows follow each other)
        u = _silu((full[:, j:j + TAPS] * s["cw"].t()).sum(1) + s["cb"])
        x = u[:, :inner].view(S, H, P)
        B = u[:, inner:inner + G * N].view(S, G, N).repeat_interleave(H // G, 1)
        C = u[:, inner + G * N:].view(S, G, N).repeat_interleave(H // G, 1)
        h = h * torch.exp(dt[:, j] * s["a"])[..., None, None] + (dt[:, j, :, None] * x)[..., None] * B[:, :, None, :]
        out.append((h * C[:, :, None, :]).sum(3) + x * s["d"][:, None])
    s["h1"][slots] = h
    s["ring"][slots[:, None], (pos[:, None] + torch.arange(each, device=pos.device)) % s["cap"]] = raw
    return {"y": torch.stack(out, 1).reshape(S * each, inner).to(DTYPE[c["io"]]), "state": s["h1"], "ring": s["ring"]}


def _rms(v):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)


def _plain_gated(c, s):
    T, D, G = c["rows"], c["width"], c["groups"]
    y, gate = s["y"].float(), _silu(s["z"].float())
    v = y if c["order"] else y * gate
    v = _rms(v.view(T, G, D // G)).view(T, D) * s["w"]
    return (v * gate if c["order"] else v).to(s["y"].dtype)


def _plain_residual(c, s):
    v = s["x"].float()
    if c["post"]:
        v = _rms(v) * s["post"]
    if c["gate"]:
        v = v * s["gate"]
    h = s["h"].float() + s["scale"] * v
    return {"stream": h.to(s["h"].dtype), "out": (_rms(h) * s["pre"]).to(s["x"].dtype)}


def _plain_q4(c, s):
    mt, kt, gr = _q4_sizes(c)
    nib, sc = s["w"][..., :1024], s["w"][..., 1024:].contiguous().view(torch.float16)
    n = torch.stack([nib & 15, nib >> 4], -1).view(mt, kt, 4, 16, 4, 2, 4)      # tile, g, m, j, e % 2, e / 2
    q = n.permute(0, 3, 1, 4, 2, 6, 5).reshape(mt * 16, kt * gr, c["group"]).float() - 8.0
    scale = sc.view(mt, kt, 4, gr, 4).permute(0, 2, 4, 1, 3).reshape(mt * 16, kt * gr, 1).float()
    w = (q * scale).view(mt * 16, kt * 128)[:c["out"], :c["in"]]
    return torch.matmul(s["x"].float(), w.t()).to(s["x"].dtype)


# ---- the framework's calls

_engine = []


def _ops():
    """The one GPU handle a program opens."""
    if not _engine:
        from nextsycl_amd import Gpu
        from nextsycl_amd.attn import Ops
        _engine.append(Ops(Gpu.open(0)))
    return _engine[0]


def _buffers(s):
    """The state's tensors as the library's buffers: a program wraps its memory once."""
    from nextsycl_amd import DevBuf
    if "b" not in s:
        s["b"] = {k: DevBuf(_ops().gpu, t.numel() * t.element_size(), _ptr=t.data_ptr(), _owner=t) for k, t in s.items() if isinstance(t, torch.Tensor)}
        s["qt"] = {"f32": 0, "f16": 1, "bf16": 2}
    return s["b"]


def _projected(c, s, n):
    """x B C and the step sizes inside the in-projection's rows."""
    b, e = _buffers(s), SIZE[c["io"]]
    if "xbc" not in b:
        H, P, N, G, inner, chan = _sizes(c)
        rows = b["rows"]
        b["xbc"] = rows.view(inner * e, rows.len - inner * e)
        b["dt"] = rows.view((inner + chan) * e, rows.len - (inner + chan) * e)
    return b


def _own_prompt(c, s):
    from nextsycl_amd import DevBuf
    ops, b = _ops(), _projected(c, s, c["rows"])
    H, P, N, G, inner, chan = _sizes(c)
    T, p0 = c["rows"], c["past"]
    if "scratch" not in s:
        s["scratch"] = DevBuf(ops.gpu, max(4, 4 * ops.ssm_prompt_scratch(T, H, P, N, G, TAPS)))
    ops.ssm_prompt(s["qt"][c["io"]], b["xbc"], s["row"], b["dt"], s["row"], b["cw"], b["cb"], b["a"], b["dtb"], b["d"], b["ring"], 8, p0, T, H, P, N, G, TAPS,
                   b.get("h0"), b["h1"], b["y"], inner, s["scratch"])
    return {"y": s["y"], "state": s["h1"], "ring": s["ring"]}


def _own_step(c, s):
    ops, b = _ops(), _projected(c, s, c["slots"] * c["each"])
    H, P, N, G, inner, chan = _sizes(c)
    ops.ssm_step(s["qt"][c["io"]], b["xbc"], s["row"], b["dt"], s["row"], b["cw"], b["cb"], b["a"], b["dtb"], b["d"], b["ring"], s["cap"], 0, c["slots"] * c["each"],
                 H, P, N, G, TAPS, b["h0"], b["h1"], b["y"], inner, nslots=s["nslots"], slots=b["slots"], pos=b["pos"])
    return {"y": s["y"], "state": s["h1"], "ring": s["ring"]}


def _own_gated(c, s):
    ops, b = _ops(), _buffers(s)
    D = c["width"]
    ops.norm_gated(s["qt"][c["io"]], b["y"], D, b["z"], D, b["w"], b["out"], D, c["rows"], D, c["groups"], EPS, c["order"])
    return s["out"]


def _own_residual(c, s):
    ops, b = _ops(), _buffers(s)
    D = c["width"]
    ops.norm_residual(s["qt"][c["io"]], s["qt"][c["stream"]], b["x"], D, b["h"], D, b["h1"], D, b["out"], D, c["rows"], D, EPS, s["scale"], post=b.get("post"),
                      gate=b.get("gate"), pre=b["pre"])
    return {"stream": s["h1"], "out": s["out"]}


def _own_q4(c, s):
    ops, b = _ops(), _buffers(s)
    ops.q4_product(s["qt"][c["io"]], b["x"], c["in"], b["w"], c["group"], b["y"], c["out"], c["rows"], c["out"], c["in"])
    return s["y"]


def run(state):
    c = state["case"]
    if own:
        return {"prompt": _own_prompt, "step": _own_step, "gated": _own_gated, "residual": _own_residual, "q4": _own_q4}[c["op"]](c, state)
    return {"prompt": _plain_prompt, "step": _plain_step, "gated": _plain_gated, "residual": _plain_residual, "q4": _plain_q4}[c["op"]](c, state)


# ---- what a pass cannot do without

def work(case):
    c, e = case, SIZE[case["io"]]
    if c["op"] in ("prompt", "step"):
        H, P, N, G, inner, chan = _sizes(c)
        seqs = 1 if c["op"] == "prompt" else c["slots"]
        rows = c["rows"] if c["op"] == "prompt" else seqs * c["each"]
        state = 4 * H * P * N * seqs * (1 if c.get("past") == 0 else 2)
        ring = 4 * chan * (TAPS - 1) * seqs * 2
        # a row's outer product into the state, the state's product with C, the decay, the taps
        return {"bytes": rows * (chan + H + inner) * e + state + ring, "flops": rows * (5 * H * P * N + 2 * TAPS * chan)}
    if c["op"] == "gated":
        return {"bytes": 3 * c["rows"] * c["width"] * e + 4 * c["width"], "flops": 8 * c["rows"] * c["width"]}
    if c["op"] == "residual":
        n = c["rows"] * c["width"]
        return {"bytes": n * (2 * e + 2 * SIZE[c["stream"]]) + 4 * c["width"] * (1 + c["post"] + c["gate"]), "flops": 8 * n}
    T, M, K = c["rows"], c["out"], c["in"]
    return {"bytes": M * K // 2 + M * ((K + c["group"] - 1) // c["group"]) * 2 + T * (M + K) * e, "flops": 2 * T * M * K}


# ---- from the definitions, in 64 bits

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "gated":
        z = s["z"].double()
        gate = z * torch.special.expit(z)
        v = (s["y"].double() * (1.0 if c["order"] else gate)).view(c["rows"], c["groups"], -1)
        v = (v * torch.rsqrt(v.square().sum(2, keepdim=True) / v.shape[2] + EPS)).reshape(c["rows"], -1) * s["w"].double()
        return v * gate if c["order"] else v
    if c["op"] == "residual":
        norm = lambda v: v * torch.rsqrt(v.square().sum(1, keepdim=True) / v.shape[1] + EPS)  # noqa: E731
        v = s["x"].double()
        v = norm(v) * s["post"].double() if c["post"] else v
        h = s["h"].double() + s["scale"] * (v * s["gate"].double() if c["gate"] else v)
        return {"stream": h, "out": norm(h) * s["pre"].double()}
    if c["op"] == "q4":
        return _exact_q4(c, s)
    return _exact_scan(c, s)


def _exact_q4(c, s):
    """Weight (m, k) looked up where the layout says it is."""
    mt, kt, gr = _q4_sizes(c)
    m = torch.arange(c["out"], device="cuda")[:, None]
    k = torch.arange(c["in"], device="cuda")[None]
    tile = (m // 16 * kt + k // 128) * (1024 + 32 * gr)
    i = k % 128
    e = i % 8
    lane, nibble = m % 16 + 16 * (i // 8 % 4), e % 2 * 4 + e // 2
    flat = s["w"].view(-1)
    q = (flat[tile + 16 * lane + 4 * (i // 32) + nibble // 2].int() >> (4 * (nibble % 2))) & 15
    at = tile + 1024 + 2 * (m % 16 // 4 * 4 * gr + i // c["group"] * 4 + m % 4)
    bits = flat[at].int() | flat[at + 1].int() << 8
    w = (q - 8).double() * bits.to(torch.int16).view(torch.float16).double()
    return s["x"].double() @ w.t()


def _exact_scan(c, s):
    """One row after another."""
    H, P, N, G, inner, chan = _sizes(c)
    prompt = c["op"] == "prompt"
    S, each = (1, c["rows"]) if prompt else (c["slots"], c["each"])
    rows = s["rows"].double().view(S, each, -1)
    ring = (s["ring"][None] if prompt else s["ring"]).double()
    slots = torch.zeros(1, dtype=torch.long, device="cuda") if prompt else s["slots"].view(S, each)[:, 0].long()
    pos = torch.full((1,), c["past"], device="cuda") if prompt else s["pos"].view(S, each)[:, 0].long()
    states = torch.zeros(1, H, P, N, dtype=torch.float64, device="cuda") if s["h0"] is None else s["h0"].double().view(-1, H, P, N)
    out, cap = (s["h1"][None] if prompt else s["h1"]).double(), ring.shape[1]
    h, y = states[slots], torch.empty(S, each, inner, dtype=torch.float64, device="cuda")
    raw = rows[..., inner:inner + chan]
    # a row's input k rows back: the pass's own rows, the ring's in front of them, nothing in front of the first position
    acc = s["cb"].double().expand(S, each, chan).clone()
    for k in range(TAPS):
        tap = s["cw"][:, TAPS - 1 - k].double()
        acc[:, k:] += tap * raw[:, :each - k]
        for t in range(min(k, each)):
            there = pos + t - k
            acc[:, t] += tap * torch.where(there[:, None] >= 0, ring[slots, there % cap], torch.zeros((), dtype=torch.float64, device="cuda"))
    u = acc * torch.special.expit(acc)
    step = torch.logaddexp(rows[..., inner + chan:] + s["dtb"].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    keep, per = torch.exp(step * s["a"].double()), H // G
    for t in range(each):
        x = u[:, t, :inner].view(S, G, per, P, 1)
        b, cc = u[:, t, inner:inner + G * N].view(S, G, 1, 1, N), u[:, t, inner + G * N:].view(S, G, 1, N, 1)
        g = h.view(S, G, per, P, N)
        g.mul_(keep[:, t].view(S, G, per, 1, 1)).add_(x * step[:, t].view(S, G, per, 1, 1) * b)
        y[:, t] = (torch.matmul(g, cc)[..., 0] + s["d"].double().view(G, per, 1) * x[..., 0]).reshape(S, inner)
    out[slots] = h
    for t in range(max(0, each - TAPS + 1) if prompt else 0, each):
        ring[slots, (pos + t) % cap] = raw[:, t]
    return {"y": y.view(S * each, inner), "state": out[0] if prompt else out, "ring": ring[0] if prompt else ring}
