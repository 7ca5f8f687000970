"""Attention over a cache of 8-bit values in blocks of tokens, each block and head with a scale of its own, for several
sequences at once, and the eviction of that cache's least attended tokens, as cases that can be timed and compared: one pass
each through the public entry points (nextsycl_amd.attn.Ops), inputs resident on the GPU.

Five kinds of pass ("op"):
  store     new tokens' key and value rows into their sequences' blocks (ns_kv8_store): the pools and the blocks' scales
  attend    a token, or a few in a row, of each of several sequences over its blocks (ns_kv8_attend); with "acc" the weight
            that every cached token received, added to what it had
  prompt    a prompt's rows over one sequence's blocks (ns_kv8_prompt)
  weights   the attention weight that a prompt's last rows give every cached token (ns_kv8_weights)
  evict     the tokens of the largest accumulated weights, the first and the last ones kept in order in fresh blocks, each
            head's own (ns_kv8_evict): pools, scales, weights, the new lengths

A pool is [blocks][key heads][block][head size], one byte a value: int8, or e4m3 ("e4m3"). A block's scale is a power of two
(float32), so a value is exactly code x scale. Pools are returned as the numbers they hold, in units of the scales beside them:
both are defined exactly, nothing in them is a matter of rounding differently."""
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# the largest code, and the exponents between which a scale is held (a value is then exactly a half)
MOST = {"int8": 127.0, "e4m3": 448.0}
HELD = {"int8": (-24, 9), "e4m3": (-15, 7)}


def listed():
    return [
        # a token of each of many chats
        {"name": "store_tokens_64", "op": "store", "form": "int8", "io": "bf16", "seqs": 64, "rows": 1, "ragged": False, "context": 2011, "kv": 8, "head": 128, "block": 64},
        # a whole prompt's rows, float32 as the projections leave them
        {"name": "store_prompt_8k", "op": "store", "form": "e4m3", "io": "f32", "seqs": 1, "rows": 8192, "ragged": False, "context": 0, "kv": 8, "head": 128, "block": 32},
        # a token of one chat
        {"name": "token_4k", "op": "attend", "form": "int8", "io": "f16", "seqs": 1, "rows": 1, "ragged": False, "context": 4095, "heads": 32, "kv": 8, "head": 128, "block": 64, "acc": False},
        # a token of each of many chats, from a few tokens long to 8000
        {"name": "tokens_64", "op": "attend", "form": "int8", "io": "bf16", "seqs": 64, "rows": 1, "ragged": True, "context": 8000, "heads": 32, "kv": 8, "head": 128, "block": 32, "acc": False},
        # a token and up to three drafts of each of three long chats, heads of 256
        {"name": "verify_43k", "op": "attend", "form": "e4m3", "io": "f32", "seqs": 3, "rows": 4, "ragged": True, "context": 43003, "heads": 24, "kv": 4, "head": 256, "block": 128, "acc": False},
        # a token of one very long chat whose tokens' weights are kept for eviction
        {"name": "token_128k_acc", "op": "attend", "form": "e4m3", "io": "f16", "seqs": 1, "rows": 1, "ragged": False, "context": 131071, "heads": 64, "kv": 4, "head": 128, "block": 64, "acc": True},
        # a whole prompt
        {"name": "prompt_8k", "op": "prompt", "form": "int8", "io": "bf16", "rows": 8192, "past": 0, "heads": 40, "kv": 8, "head": 128, "block": 64},
        # a follow-up question behind a long context, heads of 256
        {"name": "prompt_turn", "op": "prompt", "form": "e4m3", "io": "bf16", "rows": 115, "past": 20011, "heads": 16, "kv": 2, "head": 256, "block": 16},
        # the prompt's last rows as observers of all of it
        {"name": "weights_last_64", "op": "weights", "form": "int8", "io": "bf16", "rows": 64, "past": 16320, "heads": 32, "kv": 8, "head": 128, "block": 64},
        # every row of a chunk, float32
        {"name": "weights_chunk", "op": "weights", "form": "e4m3", "io": "f32", "rows": 1024, "past": 3001, "heads": 24, "kv": 4, "head": 256, "block": 32},
        # one long chat down to a quarter
        {"name": "evict_32k", "op": "evict", "form": "int8", "seqs": 1, "ragged": False, "context": 32768, "keep": 8192, "first": 4, "last": 256, "kv": 8, "head": 128, "block": 64},
        # chats of many lengths down to 512 tokens, some of them shorter than that
        {"name": "evict_ragged", "op": "evict", "form": "e4m3", "seqs": 12, "ragged": True, "context": 3001, "keep": 517, "first": 1, "last": 61, "kv": 4, "head": 256, "block": 16},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, key heads, head size)
HEADS = [(32, 8, 128), (64, 4, 128), (40, 8, 128), (16, 2, 256), (24, 4, 256), (8, 8, 128), (32, 2, 128), (10, 1, 128), (15, 5, 128), (28, 4, 128), (6, 3, 256)]


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "attend", "prompt", "weights", "evict"])
    Hq, Hkv, D = rng.choice(HEADS)
    c = {"op": op, "form": rng.choice(["int8", "e4m3"]), "kv": Hkv, "head": D, "block": rng.choice([16, 32, 64, 128])}
    values = 64 * 8000 * 8 * 128                   # of a cache, at most
    if op == "store":
        c.update(io=rng.choice(["f32", "f16", "bf16"]), seqs=rng.choice([1, _log(rng, 1, 64)]), ragged=rng.random() < 0.5, context=rng.choice([0, _log(rng, 1, 4000)]))
        c["rows"] = _log(rng, 1, max(1, 8192 * 8 * 128 // (Hkv * D * c["seqs"])))
    elif op == "attend":
        c.update(io=rng.choice(["f32", "f16", "bf16"]), heads=Hq, seqs=rng.choice([1, _log(rng, 1, 64)]), rows=rng.choice([1, 1, rng.randint(2, 8), rng.randint(9, 16)]),
                 ragged=rng.random() < 0.6, acc=rng.random() < 0.4)
        c["context"] = _log(rng, 1, min(131071, values // (4 * c["seqs"] * Hkv * D)))
    elif op == "prompt":
        c.update(io="bf16", heads=Hq, past=rng.choice([0, _log(rng, 1, 40000)]))
        c["rows"] = _log(rng, 1, max(1, min(8192, 8192 * 4096 * 40 * 128 // (Hq * D * (c["past"] + 4096)))))
    elif op == "weights":
        c.update(io=rng.choice(["f32", "f16", "bf16"]), heads=Hq, past=rng.choice([0, _log(rng, 1, 40000)]))
        c["rows"] = _log(rng, 1, max(1, min(1024, 1024 * 4096 * 24 * 256 // (Hq * D * (c["past"] + 1024)))))
    else:
        c.update(seqs=rng.choice([1, _log(rng, 1, 24)]), ragged=rng.random() < 0.5)
        c["context"] = _log(rng, 2, min(65536, 32768 * 8 * 128 * 2 // (c["seqs"] * Hkv * D)))
        c["keep"] = rng.randint(max(1, c["context"] // 16), c["context"])
        c["first"] = rng.randint(0, min(4, c["keep"]))
        c["last"] = rng.randint(0, (c["keep"] - c["first"]) // 2)
    return c


# ---- what a program has in hand before the call

class _Random:
    def __init__(self, seed):
        self.g = torch.Generator("cuda").manual_seed(seed)

    def __call__(self, *shape, sigma=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g, device="cuda") * sigma).to(dtype)

    def uniform(self, lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(*shape, generator=self.g, device="cuda")


def prepare(case, seed):
    s = {"store": _prepare_store, "attend": _prepare_attend, "prompt": _prepare_prompt, "weights": _prepare_weights, "evict": _prepare_evict}[case["op"]](case, _Random(seed))
    s["case"] = case
    torch.cuda.synchronize()      # torch's stream and the library's are two
    return s


def _channels(c, rand):
    """Some features of a head's keys are several times as large as the others; the values' are alike."""
    return torch.exp(0.6 * rand(c["kv"], 1, c["head"])), 0.5 + rand.uniform(0.0, 1.0, c["kv"], 1, 1)


def _pools(c, rand, blocks, spare):
    """Pools of `blocks` filled blocks and `spare` empty ones, and their scales."""
    Hkv, D, B, form = c["kv"], c["head"], c["block"], c["form"]
    s = {}
    for name, gain in zip(("k", "v"), _channels(c, rand)):
        rows = rand(blocks, Hkv, B, D).mul_(gain).mul_(torch.exp(0.3 * rand(blocks, Hkv, 1, 1)))
        scale = _scale(rows.abs().amax((2, 3)), form)
        codes = _codes(rows.div_(scale[..., None, None]), form)
        s[name] = torch.cat([codes, codes.new_zeros(spare, Hkv, B, D)])
        s[name + "s"] = torch.cat([scale, scale.new_ones(spare, Hkv)])
    return s


def _lengths(c, rand, most, least=1):
    """The sequences' contexts: `most` each, or anything from a few tokens up to it, spread over their logarithm."""
    S = c["seqs"]
    if not c["ragged"]:
        return torch.full((S,), most, dtype=torch.int32, device="cuda")
    spread = torch.exp(rand.uniform(math.log(max(1, most // 64)), math.log(max(1, most)), S)).round().to(torch.int32).clamp(min(least, most), most)
    spread[:1] = most
    return spread


def _tables(c, rand, lens, tmax, blocks):
    """Every sequence's blocks, anywhere in the pool; entries behind its last are no blocks."""
    S = c["seqs"]
    order = torch.argsort(rand(blocks)).to(torch.int32)[:S * tmax].view(S, tmax)
    held = torch.arange(tmax, device="cuda")[None] * c["block"] < lens[:, None]
    return torch.where(held, order, -1).to(torch.int32).contiguous()


def _starts(c):
    """Where each sequence's rows begin: `rows` of them each, or 1 .. rows (as many whatever the seed)."""
    S, n = c["seqs"], c["rows"]
    counts = 1 + (n - 1 + 5 * torch.arange(S, device="cuda") * c["ragged"]) % n
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)


def _blocks_of(tokens, B):
    return (tokens + B - 1) // B


def _prepare_store(c, rand):
    S, n, B, kind = c["seqs"], c["rows"], c["block"], DTYPE[c["io"]]
    tmax = _blocks_of(c["context"] + n, B)
    blocks = S * tmax
    s = _pools(c, rand, blocks, 0)
    s["lens"] = _lengths(c, rand, c["context"], 0)
    s["start"] = _starts(c)
    s["T"] = int(s["start"][-1])
    s["tmax"] = tmax
    s["table"] = _tables(c, rand, s["lens"] + s["start"].diff(), tmax, blocks)
    gk, gv = _channels(c, rand)
    s["krows"] = (rand(s["T"], c["kv"], c["head"]) * gk[:, 0] * 1.5).to(kind).view(s["T"], -1)
    s["vrows"] = (rand(s["T"], c["kv"], c["head"]) * gv[:, 0] * 1.5).to(kind).view(s["T"], -1)
    return s


def _prepare_attend(c, rand):
    S, n, B = c["seqs"], c["rows"], c["block"]
    tmax = _blocks_of(c["context"] + n, B)
    blocks = S * tmax
    s = _pools(c, rand, blocks, 0)
    s["lens"] = _lengths(c, rand, c["context"])
    s["start"] = _starts(c)
    s["T"], s["tmax"], s["longest"] = int(s["start"][-1]), tmax, c["context"] + n
    s["table"] = _tables(c, rand, s["lens"] + s["start"].diff(), tmax, blocks)
    s["q"] = rand(s["T"], c["heads"] * c["head"], sigma=1.3, dtype=DTYPE[c["io"]])
    s["out"] = torch.empty_like(s["q"])
    if c["acc"]:
        s["acc0"] = rand.uniform(0.0, 4.0, blocks, c["kv"], B)
        s["acc1"] = torch.zeros_like(s["acc0"])
    return s


def _one(c, rand):
    """One sequence's blocks and its rows."""
    tokens, B = c["past"] + c["rows"], c["block"]
    tmax = _blocks_of(tokens, B)
    s = _pools(c, rand, tmax + 3, 0)
    s["tmax"], s["T"] = tmax, c["rows"]
    s["table"] = torch.argsort(rand(tmax + 3)).to(torch.int32)[:tmax].contiguous()
    s["q"] = rand(c["rows"], c["heads"] * c["head"], sigma=1.3, dtype=DTYPE[c["io"]])
    return s


def _prepare_prompt(c, rand):
    s = _one(c, rand)
    s["out"] = torch.empty_like(s["q"])
    return s


def _prepare_weights(c, rand):
    s = _one(c, rand)
    s["acc0"] = rand.uniform(0.0, 4.0, s["tmax"] + 3, c["kv"], c["block"])
    s["acc1"] = torch.zeros_like(s["acc0"])
    return s


def _prepare_evict(c, rand):
    S, B = c["seqs"], c["block"]
    tmax = _blocks_of(c["context"], B)
    tokeep = _blocks_of(min(c["keep"], c["context"]), B)
    blocks = S * tmax
    s = _pools(c, rand, blocks, S * tokeep)
    s["lens"] = _lengths(c, rand, c["context"])
    s["tmax"], s["longest"] = tmax, c["context"]
    s["table"] = _tables(c, rand, s["lens"], tmax, blocks)
    s["to"] = torch.full((S, tmax), -1, dtype=torch.int32, device="cuda")
    s["to"][:, :tokeep] = blocks + torch.argsort(rand(S * tokeep)).to(torch.int32).view(S, tokeep)
    # a few tokens have most of the weight, and quite a few have none at all
    acc = torch.exp(2.0 * rand(blocks + S * tokeep, c["kv"], B))
    s["acc"] = torch.where(acc < 0.2, torch.zeros_like(acc), acc)
    s["lens1"] = torch.zeros_like(s["lens"])
    return s


# ---- the plain forms

def _scale(largest, form):
    """The least power of two s with largest <= s x the largest code, held to the form's range."""
    m, e = torch.frexp(largest)                                     # largest = m 2^e, 1/2 <= m < 1
    top, width = {"int8": (127.0 / 128.0, 7), "e4m3": (448.0 / 512.0, 9)}[form]
    e = e - width + (m > top).int()
    lo, hi = HELD[form]
    return (torch.where(largest > 0, e, lo).clamp(lo, hi) + 127 << 23).view(torch.float32)           # 2^e


def _codes(v, form):
    """Values in units of their scale, rounded to the nearest code (to even), magnitudes held to the largest."""
    v = v.clamp_(-MOST[form], MOST[form])
    return v.round_().to(torch.int8) if form == "int8" else v.to(torch.float8_e4m3fn)


def _gather(s, name, ids):
    """Blocks' values as float32: [.., Hkv, B, D]."""
    at = ids.clamp(min=0).long()
    return s[name][at].float() * s[name + "s"][at][..., None, None]


def _rows_of(c, s):
    """Every row's sequence, its number there, its position."""
    start = s["start"].long()
    r = torch.arange(s["T"], device=start.device)
    seq = torch.bucketize(r, start[1:], right=True)
    i = r - start[seq]
    return seq, i, s["lens"].long()[seq] + i


def _plain_store(c, s):
    Hkv, D, B, form = c["kv"], c["head"], c["block"], c["form"]
    seq, i, pos = _rows_of(c, s)
    blk, slot = s["table"].long()[seq, pos // B], pos % B
    first = (slot == 0) | (i == 0)                                  # one row of each block that rows go into
    tb, fresh = blk[first], (slot == 0)[first]
    for x in ("k", "v"):
        rows = s[x + "rows"].float().view(-1, Hkv, D)
        largest = torch.zeros_like(s[x + "s"]).index_reduce_(0, blk, rows.abs().amax(2), "amax")
        s0 = s[x + "s"][tb]
        s1 = _scale(largest[tb], form)
        s1 = torch.where(fresh[:, None], s1, torch.maximum(s0, s1))
        held = s[x][tb].float() * (s0 / s1)[..., None, None]        # what is there, in the blocks' new units
        held = torch.where(fresh[:, None, None, None], s[x][tb].float(), held)
        s[x][tb] = _codes(held, form)
        s[x + "s"][tb] = s1
        s[x][blk, :, slot] = _codes(rows / s[x + "s"][blk][..., None], form)
    return _pool_out(s)


def _pool_out(s):
    return {x: s[x] for x in ("k", "v", "ks", "vs")}


def _plain_attend(c, s):
    Hq, Hkv, D, B, S, n = c["heads"], c["kv"], c["head"], c["block"], c["seqs"], c["rows"]
    G, tmax = Hq // Hkv, s["tmax"]
    start, lens = s["start"].long(), s["lens"].long()
    L = tmax * B
    k = _gather(s, "k", s["table"]).transpose(1, 2).reshape(S, Hkv, L, D)
    v = _gather(s, "v", s["table"]).transpose(1, 2).reshape(S, Hkv, L, D)
    i = torch.arange(n, device=lens.device)
    live = i[None] < start.diff()[:, None]                                                          # [S][n]
    r = (start[:-1, None] + i[None]).clamp(max=s["T"] - 1)
    q = s["q"].float().view(-1, Hkv, G, D)[r]                                                       # [S][n][Hkv][G][D]
    q = q.permute(0, 2, 1, 3, 4).reshape(S, Hkv, n * G, D)
    logits = torch.matmul(q, k.transpose(2, 3).contiguous()).view(S, Hkv, n, G, L) / math.sqrt(D)
    seen = torch.arange(L, device=lens.device)[None, None] <= (lens[:, None] + i)[..., None]        # [S][n][L]
    logits = torch.where(seen[:, None, :, None], logits, torch.full((), -math.inf, device=lens.device))
    w = torch.exp(logits - logits.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(S, Hkv, n * G, L), v).view(S, Hkv, n, G, D).permute(0, 2, 1, 3, 4)      # [S][n][Hkv][G][D]
    s["out"][r[live]] = o[live].reshape(-1, Hq * D).to(s["out"].dtype)
    if not c["acc"]:
        return s["out"]
    given = (w * live[:, None, :, None, None]).sum((2, 3))                                          # [S][Hkv][L]
    end = lens + start.diff()
    _add_weights(c, s, s["table"], given, lens, end)
    return {"out": s["out"], "acc": s["acc1"]}


def _add_weights(c, s, table, given, past, end):
    """acc1 = acc0 (nothing for the tokens from `past` on) + the weights given to the tokens in front of `end`."""
    S, Hkv, L = given.shape
    at = torch.arange(L, device=given.device)
    there = (at[None] < end[:, None]).nonzero()
    sq, p = there[:, 0], there[:, 1]
    blk, slot = table.view(S, -1).long()[sq, p // c["block"]], p % c["block"]
    before = torch.where((p < past[sq])[:, None], s["acc0"][blk, :, slot], torch.zeros((), device=given.device))
    s["acc1"][blk, :, slot] = before + given[sq, :, p]


def _scores(c, s):
    """One sequence's logits [Hkv][T][G][n], masked."""
    Hq, Hkv, D, T, past = c["heads"], c["kv"], c["head"], c["rows"], c["past"]
    G, n = Hq // Hkv, past + T
    k = _gather(s, "k", s["table"]).transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
    q = s["q"].float().view(T, Hkv, G, D).permute(1, 0, 2, 3).reshape(Hkv, T * G, D)
    logits = torch.matmul(q, k.transpose(1, 2).contiguous()).view(Hkv, T, G, n) / math.sqrt(D)
    seen = torch.arange(n, device=k.device)[None] <= past + torch.arange(T, device=k.device)[:, None]
    return torch.where(seen[None, :, None], logits, torch.full((), -math.inf, device=k.device))


def _plain_prompt(c, s):
    Hq, Hkv, D, T, n = c["heads"], c["kv"], c["head"], c["rows"], c["past"] + c["rows"]
    logits = _scores(c, s)
    w = torch.exp(logits - logits.amax(-1, keepdim=True))
    v = _gather(s, "v", s["table"]).transpose(0, 1).reshape(Hkv, -1, D)[:, :n].contiguous()
    o = torch.matmul(w.view(Hkv, -1, n), v).view(Hkv, T, -1, D) / w.sum(-1, keepdim=True)
    return o.transpose(0, 1).reshape(T, Hq * D).to(s["q"].dtype)


def _plain_weights(c, s):
    logits = _scores(c, s)
    w = torch.exp(logits - logits.amax(-1, keepdim=True))
    given = (w / w.sum(-1, keepdim=True)).sum((1, 2))[None]                                          # [1][Hkv][n]
    past = torch.tensor([c["past"]], device=given.device)
    _add_weights(c, s, s["table"], given, past, past + c["rows"])
    return s["acc1"]


def _kept(c, s):
    """The kept tokens' positions in order [S][Hkv][keep], how many there are, where each goes."""
    S, Hkv, B, keep, L = c["seqs"], c["kv"], c["block"], min(c["keep"], c["context"]), s["tmax"] * c["block"]
    lens = s["lens"].long()[:, None, None]
    at = torch.arange(L, device=lens.device)
    acc = s["acc"][s["table"].clamp(min=0).long()].transpose(1, 2).reshape(S, Hkv, L)
    acc = torch.where((at < c["first"]) | (at >= lens - c["last"]), torch.full((), math.inf, device=acc.device), acc)
    acc = torch.where(at < lens, acc, torch.full((), -1.0, device=acc.device))
    best = torch.sort(acc, dim=2, descending=True, stable=True).indices[..., :keep]
    count = s["lens"].long().clamp(max=keep)
    j = torch.arange(keep, device=best.device)
    best = torch.where(j < count[:, None, None], best, L)            # (behind all others)
    return torch.sort(best, dim=2).values, count, j


def _plain_evict(c, s):
    S, Hkv, B, D, form = c["seqs"], c["kv"], c["block"], c["head"], c["form"]
    idx, count, j = _kept(c, s)
    there = (j[None, :] < count[:, None]).nonzero()                  # (sequence, place)
    sq, p = there[:, 0], there[:, 1]
    src = idx[sq, :, p]                                              # [n][Hkv]
    h = torch.arange(Hkv, device=src.device)[None]
    blk, slot = s["table"].long()[sq[:, None], src // B], src % B
    to, ts = s["to"].long()[sq, p // B], p % B
    moved = s["acc"][blk, h, slot]
    for x in ("k", "v"):
        scale = s[x + "s"][blk, h]
        s1 = torch.zeros_like(s[x + "s"]).index_reduce_(0, to, scale, "amax")
        codes = _codes(s[x][blk, h, slot].float() * (scale / s1[to])[..., None], form)
        s[x][to, :, ts] = codes
        s[x + "s"][to] = s1[to]
    s["acc"][to, :, ts] = moved
    s["lens1"][:] = s["lens"].clamp(max=c["keep"])
    return dict(_pool_out(s), acc=s["acc"], lens=s["lens1"])


# ---- the framework's calls

_engine = []


def _ops():
    """The one GPU handle a program opens."""
    if not _engine:
        from nextsycl_amd import Gpu
        from nextsycl_amd.attn import Ops
        _engine.append(Ops(Gpu.open(0)))
    return _engine[0]


def _buffers(c, s):
    """The state's tensors as the library's buffers, and its cache: a program wraps its memory once."""
    if "b" not in s:
        from nextsycl_amd import DevBuf
        from nextsycl_amd.attn import Kv8
        gpu = _ops().gpu
        s["b"] = {k: DevBuf(gpu, t.numel() * t.element_size(), _ptr=t.data_ptr(), _owner=t) for k, t in s.items() if isinstance(t, torch.Tensor)}
        b = s["b"]
        s["cache"] = Kv8({"int8": 0, "e4m3": 1}[c["form"]], s["k"].shape[0], c["kv"], c["block"], c["head"], b["k"], b["v"], b["ks"], b["vs"])
        s["qt"] = {"f32": 0, "f16": 1, "bf16": 2}.get(c.get("io"))
        if c["op"] == "attend":
            s["scratch"] = DevBuf(gpu, max(4, 4 * _ops().kv8_attend_scratch(c["seqs"], c["rows"], c["heads"], c["kv"], c["head"], s["longest"], c["acc"])))
    return s["b"]


def _own_store(c, s):
    b, w = _buffers(c, s), c["kv"] * c["head"]
    _ops().kv8_store(s["cache"], s["qt"], b["krows"], w, b["vrows"], w, s["T"], b["table"], s["tmax"], c["seqs"], c["rows"], b["lens"], start=b["start"])
    return _pool_out(s)


def _own_attend(c, s):
    b = _buffers(c, s)
    _ops().kv8_attend(s["cache"], s["qt"], b["q"], c["heads"] * c["head"], s["T"], b["table"], s["tmax"], c["seqs"], c["rows"], s["longest"], b["lens"], c["heads"], b["out"],
                      s["scratch"], start=b["start"], acc0=b.get("acc0"), acc1=b.get("acc1"))
    return {"out": s["out"], "acc": s["acc1"]} if c["acc"] else s["out"]


def _own_prompt(c, s):
    b = _buffers(c, s)
    _ops().kv8_prompt(s["cache"], s["qt"], b["q"], c["heads"] * c["head"], c["rows"], b["table"], s["tmax"], c["past"], c["heads"], b["out"])
    return s["out"]


def _own_weights(c, s):
    b = _buffers(c, s)
    _ops().kv8_weights(s["cache"], s["qt"], b["q"], c["heads"] * c["head"], c["rows"], b["table"], s["tmax"], c["past"], c["heads"], b["acc0"], b["acc1"])
    return s["acc1"]


def _own_evict(c, s):
    b = _buffers(c, s)
    _ops().kv8_evict(s["cache"], b["acc"], b["table"], s["tmax"], c["seqs"], s["longest"], b["lens"], b["lens1"], c["keep"], c["first"], c["last"], to=b["to"])
    return dict(_pool_out(s), acc=s["acc"], lens=s["lens1"])


def run(state):
    c = state["case"]
    if own:
        return {"store": _own_store, "attend": _own_attend, "prompt": _own_prompt, "weights": _own_weights, "evict": _own_evict}[c["op"]](c, state)
    return {"store": _plain_store, "attend": _plain_attend, "prompt": _plain_prompt, "weights": _plain_weights, "evict": _plain_evict}[c["op"]](c, state)


# ---- what a pass cannot do without (ragged lengths: their mean)

def _mean(c, most):
    """The mean of _lengths' spread."""
    lo = max(1, most // 64)
    return (most - lo) / math.log(most / lo) if c.get("ragged") and most > lo else most


def work(case):
    c, Hkv, D = case, case["kv"], case["head"]
    if c["op"] == "store":
        rows = c["seqs"] * (c["rows"] + 1) / 2 if c["ragged"] else c["seqs"] * c["rows"]
        return {"bytes": rows * Hkv * D * 2 * (SIZE[c["io"]] + 1) + 16 * c["seqs"] * Hkv, "flops": rows * Hkv * D * 4}
    if c["op"] == "evict":
        tokens, kept = c["seqs"] * _mean(c, c["context"]), c["seqs"] * min(c["keep"], _mean(c, c["context"]))
        return {"bytes": Hkv * (4 * tokens + 4 * kept + 4 * D * kept), "flops": Hkv * tokens * 4}
    Hq = c["heads"]
    if c["op"] == "attend":
        keys, rows = c["seqs"] * _mean(c, c["context"]), (c["rows"] + 1) / 2 if c["ragged"] else c["rows"]
        return {"bytes": keys * Hkv * (2 * D + (8 if c["acc"] else 0)) + 2 * c["seqs"] * rows * Hq * D * SIZE[c["io"]], "flops": 4 * keys * rows * Hq * D}
    T, n = c["rows"], c["past"] + c["rows"]
    pairs = Hq * (T * c["past"] + T * (T + 1) // 2)
    if c["op"] == "prompt":
        return {"bytes": 2 * n * Hkv * D + 2 * T * Hq * D * SIZE[c["io"]], "flops": 4 * D * pairs}
    return {"bytes": n * Hkv * (D + 8) + T * Hq * D * SIZE[c["io"]], "flops": 2 * D * pairs}


# ---- from the definitions, in 64 bits

def exact(case, seed):
    c, s = case, prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "prompt": _exact_one, "weights": _exact_one, "evict": _exact_evict}[c["op"]](c, s)


def _exact_scale(a, form):
    """The smallest of the scales there are under which the largest magnitude is no more than the largest code (else the largest scale)."""
    lo, hi = HELD[form]
    steps = (torch.arange(lo, hi + 1, device=a.device) + 1023 << 52).view(torch.float64)            # 2^lo .. 2^hi
    short = (a.double()[..., None] > steps * MOST[form]).sum(-1).clamp(max=hi - lo)
    return steps[short]


def _exact_round(v, form):
    """To the nearest code, to the even one between two: int8 whole numbers, e4m3 multiples of 2^(exponent - 3), exponents -6 and up."""
    v = v.clamp(-MOST[form], MOST[form])
    if form == "int8":
        return torch.round(v)
    unit = (torch.frexp(v.abs().clamp(min=2.0 ** -6)).exponent.long() - 4 + 1023 << 52).view(torch.float64)
    return torch.round(v / unit) * unit


def _exact_store(c, s):
    Hkv, D, B, form = c["kv"], c["head"], c["block"], c["form"]
    out = {}
    for x in ("k", "v"):
        rows = s[x + "rows"].double().view(-1, Hkv, D)
        pool, scale = s[x].double(), s[x + "s"].double()
        for q in range(c["seqs"]):
            a, b, p0 = int(s["start"][q]), int(s["start"][q + 1]), int(s["lens"][q])
            new, first = rows[a:b], p0 // B
            if b == a:
                continue
            n = (p0 + b - a - 1) // B - first + 1
            ids = s["table"][q, first:first + n].long()
            full = torch.zeros(n * B, Hkv, D, dtype=torch.float64, device=new.device)
            off = p0 - first * B
            full[off:off + b - a] = new
            full = full.view(n, B, Hkv, D).transpose(1, 2)
            s1 = _exact_scale(full.abs().amax((2, 3)), form)
            old = scale[ids[0]].clone()
            if off:
                s1[0] = torch.maximum(s1[0], old)
                pool[ids[0]] = _exact_round(pool[ids[0]] * (old / s1[0])[:, None, None], form)
            codes = _exact_round(full / s1[..., None, None], form).transpose(1, 2).reshape(n * B, Hkv, D)
            flat = pool[ids].transpose(1, 2).reshape(n * B, Hkv, D)
            flat[off:off + b - a] = codes[off:off + b - a]
            pool[ids] = flat.view(n, B, Hkv, D).transpose(1, 2)
            scale[ids] = s1
        out[x], out[x + "s"] = pool, scale
    return out


def _tokens(c, s, x, ids, n):
    """A sequence's first n tokens in 64 bits, [Hkv][n][D]."""
    ids = ids[:_blocks_of(n, c["block"])].long()
    v = s[x][ids].double() * s[x + "s"][ids].double()[..., None, None]
    return v.transpose(0, 1).reshape(c["kv"], -1, c["head"])[:, :n]


def _exact_attend(c, s):
    Hq, Hkv, D = c["heads"], c["kv"], c["head"]
    G = Hq // Hkv
    out = torch.empty(s["T"], Hq, D, dtype=torch.float64, device="cuda")
    acc = s["acc1"].double() if c["acc"] else None
    for q in range(c["seqs"]):
        a, b, past = int(s["start"][q]), int(s["start"][q + 1]), int(s["lens"][q])
        if b > a:
            n = past + b - a
            out[a:b], w = _exact_rows(s["q"][a:b].double().view(-1, Hkv, G, D), _tokens(c, s, "k", s["table"][q], n), _tokens(c, s, "v", s["table"][q], n), past)
            if c["acc"]:
                _exact_add(c, s, acc, s["table"][q], w, past)
    out = out.view(s["T"], -1)
    return {"out": out, "acc": acc} if c["acc"] else out


def _exact_rows(q, k, v, past):
    """Rows of one sequence, a key head after another: their outputs, and the weights that each token was given."""
    T, Hkv, G, D = q.shape
    out, given = torch.empty(T, Hkv, G, D, dtype=torch.float64, device=q.device), []
    hidden = torch.arange(k.shape[1], device=q.device)[None] > past + torch.arange(T, device=q.device)[:, None]
    for h in range(Hkv):
        per = 0.0
        for g in range(G):
            w = torch.softmax(((q[:, h, g] @ k[h].t()) * D ** -0.5).masked_fill_(hidden, -math.inf), 1)
            if v is not None:
                out[:, h, g] = w @ v[h]
            per = per + w.sum(0)
        given.append(per)
    return out.view(T, -1, D), torch.stack(given)


def _exact_add(c, s, acc, ids, w, past):
    n, B = w.shape[1], c["block"]
    p = torch.arange(n, device=w.device)
    blk, slot = ids.long()[p // B], p % B
    acc[blk, :, slot] = s["acc0"].double()[blk, :, slot] * (p < past)[:, None] + w.t()


def _exact_one(c, s):
    Hkv, n = c["kv"], c["past"] + c["rows"]
    q = s["q"].double().view(c["rows"], Hkv, -1, c["head"])
    prompt = c["op"] == "prompt"
    out, w = _exact_rows(q, _tokens(c, s, "k", s["table"], n), _tokens(c, s, "v", s["table"], n) if prompt else None, c["past"])
    if prompt:
        return out.view(c["rows"], -1)
    acc = s["acc1"].double()
    _exact_add(c, s, acc, s["table"], w, c["past"])
    return acc


def _exact_evict(c, s):
    """One sequence and head after another."""
    Hkv, D, B, form = c["kv"], c["head"], c["block"], c["form"]
    pools, scales, acc = {x: s[x].double() for x in ("k", "v")}, {x: s[x + "s"].double() for x in ("k", "v")}, s["acc"].double()
    for q in range(c["seqs"]):
        n = int(s["lens"][q])
        m = min(n, c["keep"])
        p = torch.arange(n, device="cuda")
        src = s["table"][q].long()[p // B]
        for h in range(Hkv):
            a = s["acc"][src, h, p % B]
            sure = (p < c["first"]) | (p >= n - c["last"])
            if n > c["keep"]:
                rest = p[~sure]
                rest = rest[torch.sort(-a[~sure], stable=True).indices[:m - int(sure.sum())]]
                kept = torch.cat([p[sure], rest]).sort().values
            else:
                kept = p
            to = s["to"][q].long()[torch.arange(m, device="cuda") // B]
            ts = torch.arange(m, device="cuda") % B
            for x in ("k", "v"):
                from_scale = s[x + "s"].double()[src[kept], h]
                blocks = _blocks_of(m, B)
                largest = torch.zeros(blocks * B, dtype=torch.float64, device="cuda")
                largest[:m] = from_scale
                largest = largest.view(blocks, B).amax(1)
                value = s[x].double()[src[kept], h, kept % B] * from_scale[:, None]
                pools[x][to, h, ts] = _exact_round(value / largest.repeat_interleave(B)[:m, None], form)
                scales[x][s["to"][q].long()[:blocks], h] = largest
            acc[to, h, ts] = s["acc"].double()[src[kept], h, kept % B]
    return {"k": pools["k"], "v": pools["v"], "ks": scales["k"], "vs": scales["v"], "acc": acc, "lens": None}
