"""Operators of decoding with a language model, each as a user's program calls it: attention over a key and value cache held
in 8 bits, and the rules that bend the logits before a token is picked.

  attend   queries over a cache that is complete (a clip's encoder keys and values, a long document): softmax(q K^T) V, where
           K and V are int8 codes times a scale for each block of 32 tokens and head; query heads may share a key head
  append   new tokens' keys and values go into the cache, their queries see what was there and the tokens up to their own
  write    keys and values into the cache, and read back as the values that they stand for
  adjust   penalties for tokens of the history, a bias per token, a mask of the tokens that a grammar allows -> logits
  pick     the same rules and the best token of each row

A block's scale is max|x| / 127 over the rows it holds, in f32; a code is the nearest integer to x / scale, ties to even; a
block that is not full yet is coded from its f32 rows again whenever a row joins it.  q carries 1/sqrt(head width).
"""
import math

import numpy as np
import torch

own = False

BLOCK = 32


def listed():
    return [
        # one clip's encoder keys and values (30 s) under one new token: a user who waits for the next word
        {"name": "attend_stream1", "kind": "attend", "streams": 1, "heads": 20, "kv_heads": 20, "width": 64, "queries": 1, "length": 1500, "ragged": False},
        # the same for 64 clips in lock-step: the traffic that bounds a full GPU's decoding
        {"name": "attend_streams64", "kind": "attend", "streams": 64, "heads": 20, "kv_heads": 20, "width": 64, "queries": 1, "length": 1500, "ragged": False},
        # the prompts of eight clips (a prompt holds up to 224 tokens of earlier text) over clips of different lengths, one empty
        {"name": "attend_prompts8", "kind": "attend", "streams": 8, "heads": 20, "kv_heads": 20, "width": 64, "queries": 224, "length": 1500, "ragged": True},
        # one token over long contexts, four query heads to a key head; the length ends inside a block
        {"name": "attend_long4", "kind": "attend", "streams": 4, "heads": 32, "kv_heads": 8, "width": 128, "queries": 1, "length": 65551, "ragged": False},
        # self-attention of one stream's token near the end of its cache
        {"name": "append_stream1", "kind": "append", "streams": 1, "heads": 20, "kv_heads": 20, "width": 64, "queries": 1, "start": 447},
        # 64 streams in the middle of their transcripts
        {"name": "append_streams64", "kind": "append", "streams": 64, "heads": 20, "kv_heads": 20, "width": 64, "queries": 1, "start": 200},
        # the prompts of 16 streams through self-attention in one go
        {"name": "append_prompts16", "kind": "append", "streams": 16, "heads": 20, "kv_heads": 20, "width": 64, "queries": 224, "start": 0},
        # one clip's keys and values, projected in f16
        {"name": "write_clip1_f16", "kind": "write", "streams": 1, "kv_heads": 20, "width": 64, "length": 1500, "storage": "f16", "ragged": False},
        # a batch of clips of different lengths
        {"name": "write_clips24", "kind": "write", "streams": 24, "kv_heads": 20, "width": 64, "length": 1500, "storage": "f32", "ragged": True},
        # the next token of one stream under a suppress list and penalties
        {"name": "pick_stream1", "kind": "pick", "streams": 1, "vocabulary": 51866, "history": 224, "bias_rows": 1, "masks": 1},
        # 64 streams, each in its own state of a grammar
        {"name": "pick_streams64", "kind": "pick", "streams": 64, "vocabulary": 51866, "history": 448, "bias_rows": 0, "masks": 12},
        # logits of many rows for a sampler: a large vocabulary, long histories, biases of each row's own
        {"name": "adjust_streams256", "kind": "adjust", "streams": 256, "vocabulary": 131075, "history": 4099, "bias_rows": 256, "masks": 256},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    """(query heads, key heads, width)"""
    if rng.random() < 0.5:
        h = rng.randint(1, 20)
        return h, h, rng.choice([32, 64, 64, 128])
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([2, 3, 4, 7, 8]), kv, rng.choice([64, 80, 96, 128, 128, 256])


def draw(rng):
    kind = rng.choice(["attend", "attend", "append", "append", "write", "pick", "adjust"])
    if kind in ("pick", "adjust"):
        S, V = _log_int(rng, 1, 256), _log_int(rng, 257, 131072)
        return {"kind": kind, "streams": S, "vocabulary": V, "history": _log_int(rng, 1, 4096), "bias_rows": rng.choice([0, 1, S]),
                "masks": rng.choice([0, 1, rng.randint(2, 24), S])}
    H, KV, D = _heads(rng)
    S = _log_int(rng, 1, 64)
    most = max(40, min(65536, int(1.2e8 / (S * KV * D))))  # values of K: at most twice those of 64 clips
    if kind == "write":
        return {"kind": kind, "streams": S, "kv_heads": KV, "width": D, "length": _log_int(rng, 1, max(1, min(4000, most // 2))),
                "storage": rng.choice(["f32", "f16"]), "ragged": rng.random() < 0.5}
    length = _log_int(rng, 1, most)
    queries = 1
    if rng.random() < 0.4:  # a prompt, or a few tokens that were guessed ahead; as many score products as eight prompts at most
        queries = _log_int(rng, 2, max(2, min(300, int(5.0e7 / (S * H * length) * 64 / max(64, D)))))
    if kind == "attend":
        return {"kind": kind, "streams": S, "heads": H, "kv_heads": KV, "width": D, "queries": queries, "length": length, "ragged": rng.random() < 0.5}
    start = length - 1 if queries == 1 else length // BLOCK * BLOCK
    return {"kind": kind, "streams": S, "heads": H, "kv_heads": KV, "width": D, "queries": queries, "start": start}


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _kv(gen, S, T, H, D):
    """Keys or values [S*T, H*D]: channels of unequal size, a few rows far above the others, as projections give them."""
    x = _normal(gen, S * T, H * D)
    x *= torch.exp(0.5 * _normal(gen, 1, H * D))
    x *= 1 + 3 * (torch.rand(S * T, 1, generator=gen, device="cuda") < 0.01).float()
    return x


def _lengths(case, gen):
    """Valid positions of each stream: one empty and one full stream where they differ."""
    S, n = case["streams"], case["length"]
    if not case["ragged"]:
        return torch.full((S,), n, device="cuda", dtype=torch.int64)
    lens = torch.randint(0, n + 1, (S,), generator=gen, device="cuda")
    lens[0] = n
    if S > 1:
        lens[S - 1] = 0
    return lens


def _inputs(case, seed):
    """What the case's call is given, as torch tensors on the GPU."""
    gen, S, kind = _generator(seed), case["streams"], case["kind"]
    if kind in ("pick", "adjust"):
        V, n = case["vocabulary"], case["history"]
        # tokens of the history: a few frequent ones, many rare ones, and -1 where a shorter history is padded
        ids = (V * torch.rand(n, S, generator=gen, device="cuda") ** 6).long().clamp_max(V - 1)
        ids[torch.rand(n, S, generator=gen, device="cuda") < 0.05] = -1
        words = (V + 31) // 32
        masks = None
        if case["masks"]:
            allowed = torch.rand(case["masks"], words * 32, generator=gen, device="cuda") < 0.7
            bits = allowed.view(case["masks"], words, 32).long() << torch.arange(32, device="cuda")
            masks = bits.sum(-1)
            masks = torch.where(masks >= 1 << 31, masks - (1 << 32), masks).int()
        rows = None
        if case["masks"] not in (0, 1, S):
            rows = torch.randint(0, case["masks"], (S, 1), generator=gen, device="cuda")
        bias = None
        if case["bias_rows"]:
            bias = _normal(gen, case["bias_rows"], V)
            bias = torch.where(torch.rand(case["bias_rows"], V, generator=gen, device="cuda") < 0.02, 4 * bias, torch.zeros_like(bias))
        return {"logits": 3 * _normal(gen, S, V), "ids": ids, "masks": masks, "mask_rows": rows, "bias": bias}
    KV, D = case["kv_heads"], case["width"]
    if kind == "write":
        t = torch.float16 if case["storage"] == "f16" else torch.float32
        lens = _lengths(case, gen)
        return {"k": _kv(gen, S, case["length"], KV, D).to(t), "v": _kv(gen, S, case["length"], KV, D).to(t), "lens": lens}
    H, T = case["heads"], case["queries"]
    held = case["length"] if kind == "attend" else case["start"]
    got = {"k": _kv(gen, S, held, KV, D), "v": _kv(gen, S, held, KV, D)}
    q = 1.5 / math.sqrt(D) * _normal(gen, S * T, H * D)
    if kind == "attend":
        return dict(got, q=q, lens=_lengths(case, gen))
    return dict(got, qkv=torch.cat([q, _kv(gen, S, T, KV, D), _kv(gen, S, T, KV, D)], 1))


RULES = {"repetition": 1.15, "presence": 0.3, "frequency": 0.125}


# ---- the plain forms -----------------------------------------------------------------------------------------------------

def _blocks(x, S, T, H, D):
    """[S*T, H*D] -> [S, H, blocks, 32, D] f32, zeros behind the last row"""
    x = x.float().view(S, T, H, D).permute(0, 2, 1, 3)
    x = torch.nn.functional.pad(x, (0, 0, 0, -T % BLOCK))
    return x.reshape(S, H, -1, BLOCK, D)


def _quantise(x):
    """Codes and scales of blocks [..., 32, D]; the quotient in 64 bits, where values next to a border stay on their side."""
    scale = x.abs().amax((-2, -1)) / torch.full((), 127.0, device="cuda")  # (by a number, torch multiplies with 1 / 127)
    code = (x.double() / scale.double()[..., None, None]).round().clamp(-127, 127)
    return torch.where(scale[..., None, None] > 0, code, torch.zeros_like(code)).to(torch.int8), scale


def _values(code, scale):
    """[S, H, blocks, 32, D] codes -> [S, H, positions, D] f32"""
    x = code.float() * scale[..., None, None]
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def _attend(q, K, V, limit):
    """q [S, T, H, D] over K, V [S, KV, N, D]; query (s, i) sees the positions below limit[s, i]."""
    S, T, H, D = q.shape
    KV, N = K.shape[1], K.shape[2]
    q = q.view(S, T, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(S, KV, -1, D)
    seen = torch.arange(N, device="cuda") < limit[:, None, :, None]
    score = (q @ K.transpose(-1, -2)).view(S, KV, H // KV, T, N)
    score = score.masked_fill(~seen[:, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = p.view(S, KV, -1, N) @ V
    out = out.view(S, KV, H // KV, T, D) / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(0, 3, 1, 2, 4).reshape(S * T, H * D)


def _rows(values, S):
    """[S, H, T, D] -> [S*T, H*D]"""
    return values.permute(0, 2, 1, 3).reshape(S * values.shape[2], -1)


def _adjusted(s):
    """The logits under the rules, and which tokens are allowed (None: all)."""
    x, ids = s["logits"], s["ids"].t()
    S, V = x.shape
    seen = torch.zeros(S, V + 1, device="cuda")
    seen.scatter_add_(1, torch.where(ids < 0, V, ids), torch.ones_like(ids, dtype=torch.float32))
    seen = seen[:, :V]
    there = seen > 0
    r = torch.full((), RULES["repetition"], device="cuda")
    x = torch.where(there, torch.where(x > 0, x / r, x * r), x)
    x = x - seen * RULES["frequency"] - torch.where(there, RULES["presence"], 0.0)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["masks"] is None:
        return x, None
    j = torch.arange(V, device="cuda")
    allowed = (s["masks"][:, j // 32] >> (j % 32)) & 1 != 0
    if s["mask_rows"] is not None:
        allowed = allowed[s["mask_rows"][:, 0]]
    return torch.where(allowed, x, -math.inf), allowed


def _run_plain(s):
    case = s["case"]
    kind, S = case["kind"], case["streams"]
    if kind == "adjust":
        return _adjusted(s)[0]
    if kind == "pick":
        x, allowed = _adjusted(s)
        could = ~x.isnan() if allowed is None else allowed & ~x.isnan()
        best = torch.where(could, x, -math.inf).amax(1, keepdim=True)
        j = torch.arange(x.shape[1], device="cuda")
        first = torch.where(could & (x == best), j, x.shape[1]).amin(1, keepdim=True)
        return torch.cat([torch.where(first == x.shape[1], -1, first).float(), best], 1)
    KV, D = case["kv_heads"], case["width"]
    if kind == "write":
        T = case["length"]
        there = (torch.arange(T, device="cuda") < s["lens"][:, None]).view(S * T, 1)
        k, v = (_values(*_quantise(_blocks(torch.where(there, s[n].float(), 0.0), S, T, KV, D)))[:, :, :T] for n in "kv")
        return {"k": _rows(k, S), "v": _rows(v, S)}
    H, T = case["heads"], case["queries"]
    if kind == "attend":
        q = s["q"].view(S, T, H, D)
        return _attend(q, _values(*s["kc"]), _values(*s["vc"]), s["lens"][:, None].expand(S, T))
    n = case["start"]
    first, q = n // BLOCK, s["qkv"][:, :H * D].reshape(S, T, H, D)
    read, caches = [], []
    for name, at in (("k", H * D), ("v", (H + KV) * D)):
        new = s["qkv"][:, at:at + KV * D].reshape(S, T, KV, D).permute(0, 2, 1, 3)
        rows = torch.cat([s[name + "t"][:, :, :n % BLOCK], new], 2)  # f32 rows from the open block's start on
        code, scale = _quantise(_blocks(_rows(rows, S), S, rows.shape[2], KV, D))
        codes, scales = s[name + "c"]
        codes[:, :, first:first + code.shape[2]], scales[:, :, first:first + code.shape[2]] = code, scale
        caches.append(_values(codes, scales))
        read.append(_rows(caches[-1][:, :, first * BLOCK:n + T], S))
    limit = n + 1 + torch.arange(T, device="cuda").expand(S, T)
    return {"out": _attend(q, caches[0], caches[1], limit), "k": read[0], "v": read[1]}


# ---- the framework's operators -------------------------------------------------------------------------------------------

_CTX = []


def _context():
    if not _CTX:
        import importlib

        _CTX.append(importlib.import_module("fluidaudio-web_b200").CudaContext(0))
    return _CTX[0]


class _Buffer:
    def __init__(self, ptr, shape, f16, owner=None):
        self.owner = owner  # the memory goes back to the context with it: a result keeps it
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": shape, "typestr": "<f2" if f16 else "<f4", "version": 3}


def _view(ctx, t, owner=None):
    """A tensor of the context as a torch tensor on the same memory."""
    return torch.as_tensor(_Buffer(ctx.devicePtr(t), (t.rows, t.cols), t.f16, owner), device="cuda")


def _tensor(ctx, values):
    """A tensor of the context that holds `values`, a torch tensor on the GPU."""
    if values is None:
        return None
    values = values.reshape(values.shape[0], -1)
    f16 = values.dtype == torch.float16
    t = (ctx.allocF16 if f16 else ctx.alloc)(*values.shape)
    if values.numel():
        _view(ctx, t).copy_(values)
    torch.cuda.synchronize()
    return t


class _Held:
    """What a program holds of the framework's for one case; it goes back to the context with it."""

    def __init__(self, ctx):
        self.ctx, self.tensors, self.bytes, self.caches, self.out = ctx, [], [], [], []

    def tensor(self, values):
        t = _tensor(self.ctx, values)
        if t is not None:
            self.tensors.append(t)
        return t

    def release_outputs(self):
        for t in self.out:
            self.ctx.freeTensor(t)
        self.out = []

    def give(self, t):
        self.out.append(t)
        return _view(self.ctx, t, self)

    def __del__(self):
        try:
            self.ctx.sync()
            self.release_outputs()
            for t in self.tensors:
                self.ctx.freeTensor(t)
            for b in self.bytes:
                self.ctx.freeBytes(b)
            for c in self.caches:
                self.ctx.freeKvCache8(c)
            self.ctx.trimPool(0)
        except Exception:  # the process is ending
            pass


def _prepare_own(case, x):
    ctx = _context()
    held = _Held(ctx)
    s = {"case": case, "held": held}
    S, kind = case["streams"], case["kind"]
    if kind in ("pick", "adjust"):
        mask = None
        if x["masks"] is not None:
            mask = ctx.uploadBytes(x["masks"].cpu().numpy())
            held.bytes.append(mask)
        rules = dict(RULES, history=held.tensor(x["ids"].float()), n=case["history"], bias=held.tensor(x["bias"]), mask=mask,
                     maskRows=None if x["mask_rows"] is None else held.tensor(x["mask_rows"].float()))
        return dict(s, logits=held.tensor(x["logits"]), rules=rules)
    KV, D = case["kv_heads"], case["width"]
    n = case["start"] if kind == "append" else case["length"]
    cache = ctx.kvCache8(S, n + case["queries"] if kind == "append" else n, KV, D)
    held.caches.append(cache)
    lens = held.tensor(x["lens"].float().view(S, 1)) if case.get("ragged") else None
    s.update(cache=cache, lens=lens)
    if kind == "write":
        return dict(s, k=held.tensor(x["k"]), v=held.tensor(x["v"]))
    if n:
        k, v = _tensor(ctx, x["k"]), _tensor(ctx, x["v"])
        ctx.kvWrite8(cache, k, v)
        ctx.sync()
        ctx.freeTensor(k), ctx.freeTensor(v)
        ctx.trimPool(0)
    if kind == "attend":
        return dict(s, q=held.tensor(x["q"]))
    return dict(s, qkv=held.tensor(x["qkv"]))


def _run_own(s):
    case, held = s["case"], s["held"]
    ctx, kind = held.ctx, case["kind"]
    held.release_outputs()
    if kind == "adjust":
        return held.give(ctx.adjustLogits(s["logits"], **s["rules"]))
    if kind == "pick":
        return held.give(ctx.pickAdjusted(s["logits"], **s["rules"]))
    if kind == "attend":
        return held.give(ctx.attnKv8(s["q"], s["cache"], case["heads"], case["length"], lens=s["lens"]))
    if kind == "write":
        ctx.kvWrite8(s["cache"], s["k"], s["v"], counts=s["lens"])
        k, v = ctx.kvRead8(s["cache"], 0, case["length"])
        return {"k": held.give(k), "v": held.give(v)}
    n, T = case["start"], case["queries"]
    out = held.give(ctx.attnAppendKv8(s["qkv"], s["cache"], case["heads"], n))
    first = n // BLOCK * BLOCK  # the blocks that the call changed
    k, v = ctx.kvRead8(s["cache"], first, n + T - first)
    return {"out": out, "k": held.give(k), "v": held.give(v)}


# ---- the interface -------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    x = _inputs(case, seed)
    if own:
        return _prepare_own(case, x)
    s = dict(x, case=case)
    if case["kind"] not in ("attend", "append"):
        return s
    S, KV, D = case["streams"], case["kv_heads"], case["width"]
    held = case["length"] if case["kind"] == "attend" else case["start"]
    for name in "kv":
        rows = _blocks(s.pop(name), S, held, KV, D)
        codes = _quantise(rows) if held else (rows.to(torch.int8), rows.sum((-2, -1)))
        if case["kind"] == "append":
            full, rest = held // BLOCK, held % BLOCK
            s[name + "t"] = rows[:, :, -1].clone() if rest else torch.zeros(S, KV, BLOCK, D, device="cuda")
            room = (held + case["queries"] + BLOCK - 1) // BLOCK - codes[0].shape[2]
            codes = (torch.nn.functional.pad(codes[0], (0, 0, 0, 0, 0, room)), torch.nn.functional.pad(codes[1], (0, room)))
        s[name + "c"] = tuple(c.contiguous() for c in codes)
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    S, kind = case["streams"], case["kind"]
    if kind in ("pick", "adjust"):
        V = case["vocabulary"]
        bytes_ = 4.0 * S * V * (2 if kind == "adjust" else 1) + 4.0 * S * case["history"] + 4.0 * case["bias_rows"] * V + case["masks"] * ((V + 31) // 32) * 4.0
        return {"bytes": bytes_ + (8.0 * S if kind == "pick" else 0), "flops": 6.0 * S * V}
    KV, D = case["kv_heads"], case["width"]
    code = lambda rows: 2.0 * S * KV * (rows * D + 4 * ((rows + BLOCK - 1) // BLOCK))  # noqa: E731  K and V in 8 bits
    if kind == "write":
        T = case["length"]
        return {"bytes": 2.0 * S * T * KV * D * (2 if case["storage"] == "f16" else 4) + 2 * code(T) + 8.0 * S * T * KV * D, "flops": 4.0 * S * T * KV * D}
    H, T = case["heads"], case["queries"]
    ends = 4.0 * S * T * 2 * H * D  # queries in, results out
    if kind == "attend":
        return {"bytes": code(case["length"]) + ends, "flops": 4.0 * S * T * H * D * case["length"]}
    n = case["start"]
    changed = n + T - n // BLOCK * BLOCK  # rows of the blocks that change: coded and given back as values
    return {"bytes": code(n + T) + code(changed) + ends + 8.0 * S * KV * D * (T + n % BLOCK + changed), "flops": 4.0 * S * H * D * (T * n + T * (T + 1) / 2)}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------

def _stored64(x):
    """What rows [T, D] of one head are stored as: block by block, the scale being an f32 by definition."""
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    T = x.shape[0]
    full = T // BLOCK * BLOCK
    for part, rows in ((x[:full].double().reshape(-1, BLOCK * x.shape[1]), slice(0, full)), (x[full:].double().reshape(-1, (T - full) * x.shape[1]) if T > full else None, slice(full, T))):
        if part is None or not part.numel():
            continue
        step = (part.abs().max(1).values / 127).float().double().unsqueeze(1)
        code = torch.where(step > 0, torch.round(part / step.clamp_min(1e-300)), torch.zeros_like(part))
        out[rows] = (code.clamp(-127, 127) * step).reshape(-1, x.shape[1])
    return out


def exact(case, seed):
    x = _inputs(case, seed)
    S, kind = case["streams"], case["kind"]
    if kind in ("pick", "adjust"):
        V = case["vocabulary"]
        best, rows = [], []
        r = {k: float(np.float32(v)) for k, v in RULES.items()}
        for s in range(S):
            y = x["logits"][s].double()
            used = x["ids"][:, s]
            c = torch.bincount(used[used >= 0], minlength=V).double()
            y = torch.where(c > 0, torch.where(y > 0, y / r["repetition"], y * r["repetition"]) - r["presence"], y) - c * r["frequency"]
            if x["bias"] is not None:
                y = y + x["bias"][s if case["bias_rows"] > 1 else 0].double()
            if x["masks"] is not None:
                m = int(x["mask_rows"][s, 0]) if x["mask_rows"] is not None else (s if case["masks"] > 1 else 0)
                bits = np.unpackbits(x["masks"][m].cpu().numpy().view(np.uint8), bitorder="little")[:V]
                y[torch.from_numpy(bits == 0).cuda()] = -math.inf
            rows.append(y)
            if kind == "pick":
                top = float(y.max())
                where = torch.nonzero(y == top)
                best.append([float(where[0, 0]) if top > -math.inf else -1.0, top])
        return torch.stack(rows) if kind == "adjust" else torch.tensor(best, dtype=torch.float64)
    KV, D = case["kv_heads"], case["width"]
    if kind == "write":
        T = case["length"]
        got = {n: torch.zeros(S * T, KV * D, dtype=torch.float64, device="cuda") for n in "kv"}
        for s in range(S):
            for h in range(KV):
                for n in "kv":
                    length = int(x["lens"][s])
                    got[n][s * T:s * T + length, h * D:(h + 1) * D] = _stored64(x[n][s * T:s * T + length, h * D:(h + 1) * D])
        return got
    H, T = case["heads"], case["queries"]
    held = case["length"] if kind == "attend" else case["start"]
    total = held if kind == "attend" else held + T
    first = held // BLOCK * BLOCK
    q = (x["q"] if kind == "attend" else x["qkv"][:, :H * D]).double().view(S, T, H, D)
    out = torch.zeros(S, T, H, D, dtype=torch.float64, device="cuda")
    read = {n: torch.zeros(S, total - first, KV * D, dtype=torch.float64, device="cuda") for n in "kv"}
    for s in range(S):
        for h in range(KV):
            stored = {}
            for n, at in (("k", H * D), ("v", (H + KV) * D)):
                rows = x[n][s * held:(s + 1) * held, h * D:(h + 1) * D]
                if kind == "append":
                    rows = torch.cat([rows, x["qkv"][s * T:(s + 1) * T, at + h * D:at + (h + 1) * D]])
                stored[n] = _stored64(rows)
                if kind == "append":
                    read[n][s, :, h * D:(h + 1) * D] = stored[n][first:]
            for j in range(h * (H // KV), (h + 1) * (H // KV)):
                z = q[s, :, j] @ stored["k"].t()
                if kind == "append":
                    z = torch.where(torch.ones_like(z, dtype=torch.bool).tril(held), z, -math.inf)
                else:
                    z = z[:, :int(x["lens"][s])]
                if z.shape[1]:
                    out[s, :, j] = torch.softmax(z, 1) @ stored["v"][:z.shape[1]]
    out = out.reshape(S * T, H * D)
    return out if kind == "attend" else {"out": out, "k": read["k"].reshape(-1, KV * D), "v": read["v"].reshape(-1, KV * D)}
