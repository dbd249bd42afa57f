"""Cases and plain forms of the sequence operators: attention over packed sequences (forward, backward), the append to a paged
key / value cache with the rotation of positions, and attention of new tokens over such a cache.

Layouts.  Packed tensors hold the rows of all sequences one behind the other, [rows, heads, head_dim]; sequence b owns the rows
cu[b] .. cu[b + 1].  Query head h reads key / value head h // (heads // kv_heads).  A cache is two tensors
[pages, kv_heads, page_size, head_dim]; position p of sequence b lives in page table[b, p // page_size] at p % page_size.  The rotation
table is [positions, head_dim] in 32 bits: the cosines of the head_dim / 2 angles, then their sines; channel i turns with
channel i + head_dim / 2.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases --------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a handful of short utterances in the framework's own width (4 heads of 64) and type: the smallest batch of a training rank
        {"name": "packed fwd, 4 short, f32", "op": "packed", "type": "f32", "seqs": 4, "len": 101, "heads": 4, "kv_heads": 4, "dim": 64, "causal": True},
        # sixteen ragged texts / frame sequences, every key visible: an encoder's attention without its padding
        {"name": "packed fwd, 16 ragged, f16", "op": "packed", "type": "f16", "seqs": 16, "len": 800, "heads": 4, "kv_heads": 4, "dim": 64, "causal": False},
        # whole prompts, grouped heads, causal: four sequences of up to 4096
        {"name": "packed fwd, prompts, bf16", "op": "packed", "type": "bf16", "seqs": 4, "len": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True},
        # the backward pass of 32 utterances of up to 400 reduced frames (the training benchmark's batch) in 32 bits
        {"name": "packed bwd, 32 ragged, f32", "op": "grad", "type": "f32", "seqs": 32, "len": 400, "heads": 4, "kv_heads": 4, "dim": 64, "causal": True},
        # the backward pass of packed training sequences with grouped heads
        {"name": "packed bwd, long, bf16", "op": "grad", "type": "bf16", "seqs": 4, "len": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True},
        # one decoding step of eight sequences: one new token each, latency counts
        {"name": "append, 8 tokens, bf16", "op": "append", "type": "bf16", "seqs": 8, "len": 1, "context": 1500, "page": 16, "heads": 32, "kv_heads": 8, "dim": 128},
        # the prompts of a batch go into the cache, chunks of up to 2048 behind what is there
        {"name": "append, prompts, bf16", "op": "append", "type": "bf16", "seqs": 16, "len": 2048, "context": 4096, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128},
        # one sequence of moderate length decodes alone
        {"name": "decode, 1 x 1000, f16", "op": "paged", "type": "f16", "seqs": 1, "len": 1, "context": 1000, "page": 16, "heads": 4, "kv_heads": 4, "dim": 64},
        # a serving batch decodes: 64 ragged contexts of up to 4096
        {"name": "decode, 64 ragged, bf16", "op": "paged", "type": "bf16", "seqs": 64, "len": 1, "context": 4096, "page": 16, "heads": 32, "kv_heads": 8, "dim": 128},
        # two long documents: few rows, a long axis
        {"name": "decode, 2 x 100000, bf16", "op": "paged", "type": "bf16", "seqs": 2, "len": 1, "context": 100003, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128},
        # a few new tokens for each sequence (a draft that is verified, frames that stream in)
        {"name": "chunk, 16 x 5, f16", "op": "paged", "type": "f16", "seqs": 16, "len": 5, "context": 2000, "page": 32, "heads": 16, "kv_heads": 4, "dim": 64},
        # prompts that are taken in chunks of up to 512 over what the cache holds
        {"name": "chunk, 8 x 512, bf16", "op": "paged", "type": "bf16", "seqs": 8, "len": 512, "context": 6000, "page": 64, "heads": 32, "kv_heads": 8, "dim": 128},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))
    op = rng.choice(["packed", "packed", "grad", "grad", "append", "paged", "paged", "paged"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    dim = rng.choice([64, 64, 80, 96, 128, 128])
    c = {"op": op, "type": kind, "seqs": log(1, 64), "heads": heads, "kv_heads": kv_heads, "dim": dim}
    if op in ("packed", "grad"):
        most = (1 << 30) if op == "packed" else (1 << 28)          # pairs of a query head's row and a key, sequences padded to the longest
        if kind == "f32":
            most >>= 3
        longest = int(math.sqrt(most / (c["seqs"] * heads)))
        return {**c, "len": log(1, min(4096, longest)), "causal": rng.random() < 0.7}
    c["page"] = rng.choice([16, 32, 64, 128])
    row = (heads + 2 * kv_heads) * dim * SIZE[kind]
    if op == "append":
        c["len"] = log(1, max(1, min(2048, (1 << 28) // (2 * c["seqs"] * row))))
        return {**c, "context": log(1, max(1, min(4096, (1 << 29) // (c["seqs"] * row))))}
    c["len"] = rng.choice([1, 1, log(2, 16), log(17, 600)])
    key = 2 * kv_heads * dim * SIZE[kind]
    c["context"] = log(1, max(1, min(100000, (1 << 29) // (c["seqs"] * key), (1 << 28) // (c["seqs"] * heads * c["len"]))))
    return c


def _ragged(n, longest, salt):
    """n lengths of 1 .. longest, the longest among them."""
    r = random.Random(n * 1000003 + longest * 31 + salt)
    v = [r.randint(1, longest) for _ in range(n)]
    v[r.randrange(n)] = longest
    return v


def _sizes(c):
    """(new rows of each sequence, rows in the cache before them)"""
    new = _ragged(c["seqs"], c["len"], 1)
    return new, (_ragged(c["seqs"], c["context"], 2) if "context" in c else [0] * c["seqs"])


def work(c):
    new, ctx = _sizes(c)
    e, D, H, G = SIZE[c["type"]], c["dim"], c["heads"], c["kv_heads"]
    rows = sum(new)
    q, kv = rows * H * D * e, rows * G * D * e
    if c["op"] == "append":
        return {"bytes": 2 * q + 4 * kv + rows * D * 4, "flops": 3 * rows * (H + G) * D}
    if c["op"] == "paged":
        pairs = sum(n * x + n * (n + 1) // 2 for n, x in zip(new, ctx))
        return {"bytes": 2 * q + 2 * sum(n + x for n, x in zip(new, ctx)) * G * D * e, "flops": 4 * D * H * pairs}
    pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in new)
    if c["op"] == "packed":
        return {"bytes": 2 * q + 2 * kv + rows * H * 4, "flops": 4 * D * H * pairs}
    return {"bytes": 4 * q + 4 * kv + rows * H * 4, "flops": 10 * D * H * pairs}


# ---- inputs -------------------------------------------------------------------------------------------------------------------------
def _starts(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)


def _rotation(positions, dim):
    ang = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * (10000.0 ** (-torch.arange(dim // 2, device=DEV, dtype=torch.float64) * 2 / dim))
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def prepare(case, seed):
    c, t = case, TYPES[case["type"]]
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(t)

    new, ctx = _sizes(c)
    rows, D, H, G = sum(new), c["dim"], c["heads"], c["kv_heads"]
    s = {"case": c, "rows": rows, "most_new": max(new), "cu": _starts(new), "scale": D ** -0.5, "q": normal(rows, H, D)}
    if c["op"] in ("packed", "grad"):
        s["k"], s["v"] = normal(rows, G, D), normal(rows, G, D)
        s["out"], s["lse"] = torch.empty_like(s["q"]), torch.empty(H, rows, device=DEV)
        if c["op"] == "grad":                # what the forward pass has left: its output and its rows' log-sums
            s["out"], s["lse"] = _packed(s)
            s["dout"] = normal(rows, H, D)
            s["dq"], s["dk"], s["dv"] = (torch.empty_like(s[n]) for n in "qkv")
        return s
    P = c["page"]
    total = [n + x for n, x in zip(new, ctx)]
    held = [-(-n // P) for n in total]
    s["most"], width = max(total), max(held)
    pages = sum(held) + 3                     # a pool with a few pages to spare; the sequences' pages lie in it in any order
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    first, table = 0, torch.full((c["seqs"], width), -1, dtype=torch.int32, device=DEV)
    for b, n in enumerate(held):
        table[b, :n] = order[first:first + n]
        first += n
    s["table"], s["ctx"] = table, torch.tensor(ctx, dtype=torch.int32, device=DEV)
    s["kc"], s["vc"] = normal(pages, G, P, D), normal(pages, G, P, D)
    if c["op"] == "append":
        s["k"], s["v"], s["rot"] = normal(rows, G, D), normal(rows, G, D), _rotation(width * P, D)
    s["out"] = torch.empty_like(s["q"])       # the rotated queries of an append, the result of an attention
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------------------------
def _owners(s):
    """For every packed row its sequence and its place in it."""
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    b = torch.repeat_interleave(torch.arange(len(n), device=DEV), n, output_size=s["rows"])
    return b, torch.arange(s["rows"], device=DEV) - s["cu"].long()[b]


def _padded(x, s):
    """[rows, heads, dim] -> [seqs, longest, heads, dim] in 32 bits; what is behind a sequence's end is some other row."""
    at = s["cu"].long()[:-1, None] + torch.arange(s["most_new"], device=DEV)
    return x[at.clamp_(max=x.shape[0] - 1)].float()


def _by_group(x, G):
    """[seqs, n, heads, dim] -> [seqs * kv_heads, (heads / kv_heads) * n, dim]"""
    B, n, H, D = x.shape
    return x.reshape(B, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B * G, (H // G) * n, D)


def _from_group(x, B, H, b, i):
    """The inverse, packed: [seqs * kv_heads, (heads / kv_heads) * n, dim] -> [rows, heads, dim]"""
    return x.reshape(B, H, -1, x.shape[-1])[b, :, i]


def _seen(s, n_keys):
    """[seqs, 1, 1, longest, n_keys]: whether the row may look at the key"""
    i = torch.arange(s["most_new"], device=DEV)
    n = (s["cu"][1:] - s["cu"][:-1]).long()[:, None]
    if "table" in s:
        last = s["ctx"].long()[:, None] + i + 1
    else:
        last = (i + 1).expand(len(n), -1).minimum(n) if s["case"]["causal"] else n.expand(-1, len(i))
    return (torch.arange(n_keys, device=DEV) < last[:, :, None])[:, None, None]


def _logits(s, q, k, B, G):
    """Scaled products with the masked ones at minus infinity, [seqs, kv_heads, group, longest, keys]"""
    x = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(s["scale"])
    x = x.view(B, G, -1, s["most_new"], k.shape[1])
    return x.masked_fill_(~_seen(s, k.shape[1]), -math.inf)


def _attend(s, k, v):
    """The rows of s["q"] over keys and values [seqs * kv_heads, keys, dim]: the result and the rows' log-sums, in 32 bits"""
    c = s["case"]
    B, H, G = c["seqs"], c["heads"], c["kv_heads"]
    b, i = _owners(s)
    x = _logits(s, _by_group(_padded(s["q"], s), G), k, B, G)
    m = x.amax(-1, keepdim=True)
    x.sub_(m).exp_()
    l = x.sum(-1, keepdim=True)
    y = torch.matmul(x.view(B * G, -1, k.shape[1]), v).div_(l.view(B * G, -1, 1))
    return _from_group(y, B, H, b, i), (m + l.log()).view(B, H, -1)[b, :, i].t()


def _keys(s, x):
    return _padded(x, s).permute(0, 2, 1, 3).reshape(-1, s["most_new"], x.shape[-1])


def _packed(s):
    out, lse = _attend(s, _keys(s, s["k"]), _keys(s, s["v"]))
    return out.to(s["q"].dtype), lse.contiguous()


def _grad(s):
    c, t = s["case"], s["q"].dtype
    B, H, G = c["seqs"], c["heads"], c["kv_heads"]
    b, i = _owners(s)
    q, k, v = _by_group(_padded(s["q"], s), G), _keys(s, s["k"]), _keys(s, s["v"])
    # rows behind a sequence's end belong to another one: their gradient is nothing
    live = (torch.arange(s["most_new"], device=DEV) < (s["cu"][1:] - s["cu"][:-1])[:, None])[:, :, None, None]
    do = _by_group(_padded(s["dout"], s) * live, G)
    rest = torch.zeros(B, H, s["most_new"], device=DEV)
    rest[b, :, i] = s["lse"].t()
    p = _logits(s, q, k, B, G).sub_(rest.view(B, G, H // G, -1, 1)).exp_().view(B * G, -1, k.shape[1])
    dv = torch.matmul(p.transpose(1, 2).contiguous(), do)
    dp = torch.matmul(do, v.transpose(1, 2).contiguous())
    ds = p.mul_(dp.sub_((p * dp).sum(-1, keepdim=True))).mul_(s["scale"])
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(1, 2).contiguous(), q)
    return _from_group(dq, B, H, b, i).to(t), _from_group(dk, B, G, b, i).to(t), _from_group(dv, B, G, b, i).to(t)


def _turned(x, cos, sin):
    """The rotation in 32 bits, rounded once"""
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _append(s):
    b, i = _owners(s)
    at, P = s["ctx"].long()[b] + i, s["case"]["page"]
    cos, sin = s["rot"][at][:, None].chunk(2, -1)
    page = s["table"][b, at // P].long()
    s["kc"][page, :, at % P] = _turned(s["k"], cos, sin)
    s["vc"][page, :, at % P] = s["v"]
    return s["kc"], s["vc"], _turned(s["q"], cos, sin)


def _paged(s):
    at = s["table"].clamp(min=0).long()

    def held(x):
        return x[at].permute(0, 2, 1, 3, 4).reshape(s["case"]["seqs"] * x.shape[1], -1, x.shape[-1]).float()
    return _attend(s, held(s["kc"]), held(s["vc"]))[0].to(s["q"].dtype)


# ---- the framework's operators ------------------------------------------------------------------------------------------------------
_engine = None


def _handles(s):
    """The engine of the program and the framework's names for the arrays of a state: the same memory, wrapped once, as a program has it."""
    global _engine
    import numpy as np
    from vaenar_tts_amd._lib import DeviceArray, Engine
    if _engine is None:
        from vaenar_tts_amd.configs import LJHPS
        _engine = Engine(LJHPS, torch.cuda.current_device())
    if "handles" not in s:
        # bfloat16 has no NumPy type: its bits go as uint16
        kinds = {torch.float32: np.float32, torch.float16: np.float16, torch.bfloat16: np.uint16, torch.int32: np.int32}
        s["handles"] = {n: DeviceArray(_engine, x.shape, kinds[x.dtype], ptr=x.data_ptr(), owner=x) for n, x in s.items() if isinstance(x, torch.Tensor)}
    return _engine, s["handles"]


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"packed": _packed, "grad": _grad, "append": _append, "paged": _paged}[op](s)
    from vaenar_tts_amd import sequence
    e, a = _handles(s)
    if op == "packed":
        sequence.packed_attention(e, a["q"], a["k"], a["v"], a["cu"], causal=s["case"]["causal"], scale=s["scale"], out=a["out"], lse=a["lse"])
        return s["out"], s["lse"]
    if op == "grad":
        sequence.packed_attention_grad(e, a["dout"], a["q"], a["k"], a["v"], a["out"], a["lse"], a["cu"], causal=s["case"]["causal"], scale=s["scale"],
                                       dq=a["dq"], dk=a["dk"], dv=a["dv"])
        return s["dq"], s["dk"], s["dv"]
    if "cache" not in s:
        s["cache"] = sequence.PagedCache(e, a["kc"], a["vc"])
    if op == "append":
        s["cache"].append(a["k"], a["v"], a["cu"], a["ctx"], a["table"], rotation=a["rot"], q=a["q"], q_out=a["out"])
        return s["kc"], s["vc"], s["out"]
    s["cache"].attend(a["q"], a["cu"], a["ctx"], a["table"], max_new=s["most_new"], max_context=s["most"], scale=s["scale"], out=a["out"])
    return s["out"]


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------
def _exact_head(q, k, v, first, scale):
    """softmax(q k' scale) v of one head, in which row i sees the keys before first + i + 1 (all of them where first is None)"""
    x = (q @ k.t()) * scale
    if first is not None:
        x = x + torch.triu(torch.full_like(x, -math.inf), diagonal=first + 1)
    p = torch.softmax(x, -1)
    return p, torch.logsumexp(x, -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    new, ctx = _sizes(c)
    G, group = c["kv_heads"], c["heads"] // c["kv_heads"]
    if c["op"] == "append":
        kc, vc, q = s["kc"].double(), s["vc"].double(), s["q"].double()
        turn = s["rot"].double()
        half = c["dim"] // 2
        row = 0
        for b, n in enumerate(new):
            at = torch.arange(ctx[b], ctx[b] + n, device=DEV)
            # (x1 + i x2) (cos + i sin)
            z = torch.complex(turn[at, :half], turn[at, half:])[:, None]
            pages = s["table"][b].long()[torch.div(at, c["page"], rounding_mode="floor")]
            k = s["k"][row:row + n].double()
            kz = torch.complex(k[..., :half].contiguous(), k[..., half:].contiguous()) * z
            qz = torch.complex(q[row:row + n, :, :half].contiguous(), q[row:row + n, :, half:].contiguous()) * z
            kc[pages, :, at % c["page"]] = torch.cat([kz.real, kz.imag], -1)
            vc[pages, :, at % c["page"]] = s["v"][row:row + n].double()
            q[row:row + n] = torch.cat([qz.real, qz.imag], -1)
            row += n
        return kc, vc, q
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(c["heads"], s["rows"], dtype=torch.float64, device=DEV)
    dq, dk, dv = (torch.zeros(s[n].shape, dtype=torch.float64, device=DEV) if n in s else None for n in "qkv")
    row = 0
    for b, n in enumerate(new):
        r = slice(row, row + n)
        row += n
        if "table" in s:
            pages = s["table"][b].long()[: -(-(n + ctx[b]) // c["page"])]
        for h in range(c["heads"]):
            g = h // group
            if "table" in s:
                k, v = (s[x][pages, g].reshape(-1, c["dim"])[: n + ctx[b]].double() for x in ("kc", "vc"))
            else:
                k, v = s["k"][r, g].double(), s["v"][r, g].double()
            q = s["q"][r, h].double()
            first = ctx[b] if c.get("causal", True) else None
            p, l = _exact_head(q, k, v, first, s["scale"])
            out[r, h], lse[h, r] = p @ v, l
            if c["op"] == "grad":
                do = s["dout"][r, h].double()
                dv[r, g] += p.t() @ do
                dp = do @ v.t()
                ds = p * (dp - (dp * p).sum(-1, keepdim=True)) * s["scale"]
                dq[r, h] = ds @ k
                dk[r, g] += ds.t() @ q
    return {"packed": (out, lse), "grad": (dq, dk, dv), "paged": out}[c["op"]]
