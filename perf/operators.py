"""The serving operators over a paged key-value cache, measured case by case.

Four operators make one serving step of several sequences: the q|k|v rows of
new tokens are normalised, rotated and appended to a paged cache
(``kv_append_paged``), a whole batch of prompts attends over itself
(``attn_prefill_packed``), one new token per sequence attends over the cache
(``attn_decode_paged``), and the next token is drawn from the logits
(``sample``).  With ``own`` false ``run`` computes them with elementary torch
operations in 32 bits; with ``own`` true it makes the framework's calls.
"""
import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_MASK32 = 0xFFFFFFFF


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # -- append: one decode step of a single sequence (latency only)
        dict(name="append one token", op="append", tokens=1, seqs=1, ctx=1091, n_heads=8, n_kv=1, hd=256, rot=256,
             norm=True, src="f32", cache="f16", page=16, layout="head"),
        # -- append: one decode step of a full batch behind the f16 GEMM projections
        dict(name="append 256 sequences", op="append", tokens=256, seqs=256, ctx=1091, n_heads=8, n_kv=1, hd=256,
             rot=256, norm=True, src="f16", cache="f16", page=16, layout="head"),
        # -- append: the packed prompts of a prefill step, grouped heads, pages laid out token by token
        dict(name="append packed prompts", op="append", tokens=16133, seqs=16, ctx=0, n_heads=32, n_kv=8, hd=128,
             rot=128, norm=False, src="bf16", cache="bf16", page=32, layout="token"),
        # -- decode: a single sequence at the context of the decode benchmark
        dict(name="decode one sequence", op="decode", seqs=1, ctx=1091, spread=0.0, n_heads=8, n_kv=1, hd=256,
             window=0, cache="f16", page=16, layout="head"),
        # -- decode: a single very long conversation: all the work is along one axis
        dict(name="decode long context", op="decode", seqs=1, ctx=130001, spread=0.0, n_heads=8, n_kv=1, hd=256,
             window=0, cache="f16", page=64, layout="head"),
        # -- decode: a serving batch with ragged contexts and grouped heads
        dict(name="decode ragged batch", op="decode", seqs=96, ctx=4096, spread=0.9, n_heads=32, n_kv=8, hd=128,
             window=0, cache="bf16", page=32, layout="token"),
        # -- decode: a large batch of a sliding-window layer
        dict(name="decode windowed batch", op="decode", seqs=256, ctx=2000, spread=0.7, n_heads=8, n_kv=1, hd=256,
             window=512, cache="f16", page=16, layout="head"),
        # -- prefill: the prompt of the prefill benchmark
        dict(name="prefill one prompt", op="prefill", seqs=1, tokens=1024, spread=0.0, n_heads=8, n_kv=1, hd=256,
             window=0, dtype="f16"),
        # -- prefill: prompts of different lengths packed into one batch, grouped heads
        dict(name="prefill packed prompts", op="prefill", seqs=8, tokens=8003, spread=0.8, n_heads=32, n_kv=8, hd=128,
             window=0, dtype="bf16"),
        # -- prefill: one long document
        dict(name="prefill long prompt", op="prefill", seqs=1, tokens=15001, spread=0.0, n_heads=8, n_kv=1, hd=256,
             window=0, dtype="f16"),
        # -- sampling: the next token of one sequence over the whole vocabulary
        dict(name="sample one row", op="sample", rows=1, vocab=262144, logits="f32", mix="nucleus"),
        # -- sampling: a serving batch in which every request brings settings of its own
        dict(name="sample batch", op="sample", rows=128, vocab=262144, logits="f32", mix="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, most):
    """(query heads, key-value heads) with groups of one to 16, odd ones too."""
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 8, 8, 12, 16])
    n_kv = rng.choice([1, 1, 2, 3, 4, 8])
    while n_kv > 1 and group * n_kv > most:
        n_kv -= 1
    return group * n_kv, n_kv


def draw(rng):
    op = rng.choice(["append", "decode", "prefill", "sample"])
    if op == "append":
        hd = rng.choice([64, 128, 256, 256, 512])
        nh, nkv = _heads(rng, 40)
        tokens = _log(rng, 1, 16000 * 48 * 128 / ((nh + 2 * nkv) * hd) + 1)
        tokens = max(1, min(tokens, 16000))
        seqs = tokens if rng.random() < 0.5 and tokens <= 1024 else _log(rng, 1, min(tokens, 64))
        return dict(op="append", tokens=tokens, seqs=seqs, ctx=rng.randrange(0, 3000) if seqs == tokens else
                    rng.choice([0, 0, rng.randrange(1, 500)]), n_heads=nh, n_kv=nkv, hd=hd,
                    rot=rng.choice([hd, hd, hd // 2]), norm=rng.random() < 0.5, src=rng.choice(["f16", "bf16", "f32"]),
                    cache=rng.choice(["f16", "bf16"]), page=rng.choice([1, 16, 16, 32, 64, 128]),
                    layout=rng.choice(["head", "token"]))
    if op == "decode":
        hd = rng.choice([64, 128, 128, 256, 256, 512])
        nh, nkv = _heads(rng, 64)
        keys = _log(rng, 1, 400000000 // (nkv * hd))  # cached keys of the whole batch
        seqs = max(1, min(_log(rng, 1, 384), keys))
        return dict(op="decode", seqs=seqs, ctx=max(1, min(130000, keys // seqs)), spread=rng.choice([0.0, 0.5, 0.95]),
                    n_heads=nh, n_kv=nkv, hd=hd, window=rng.choice([0, 0, 0, 100, 512, 1024]),
                    cache=rng.choice(["f16", "bf16"]), page=rng.choice([1, 16, 16, 32, 64, 128]),
                    layout=rng.choice(["head", "token"]))
    if op == "prefill":
        hd = rng.choice([64, 128, 256])
        nh, nkv = _heads(rng, 32)
        seqs = _log(rng, 1, 48)
        most = min(12000, int(math.sqrt(6e8 * seqs / nh)))  # the plain form's scores stay a few GB
        tokens = max(seqs, _log(rng, 1, most))
        return dict(op="prefill", seqs=seqs, tokens=tokens, spread=rng.choice([0.0, 0.4, 0.8]), n_heads=nh, n_kv=nkv,
                    hd=hd, window=rng.choice([0, 0, 0, 128, 512, 777]), dtype=rng.choice(["f16", "bf16"]))
    vocab = _log(rng, 1000, 262144)
    return dict(op="sample", rows=max(1, min(_log(rng, 1, 300), 33000000 // vocab)), vocab=vocab,
                logits=rng.choice(["f32", "f16", "bf16"]), mix=rng.choice(["nucleus", "mixed", "plain", "topk"]))


# ------------------------------------------------------------------ inputs

def _lengths(total, n, spread):
    """n lengths of about total / n tokens, the same for a case whatever its seed: a fixed
    spiral of weights between 1 - spread and 1 + spread, at least one token each."""
    w = [1.0 + spread * math.sin(2.4 * i + 0.7) for i in range(n)]
    lens = [max(1, int(total * x / sum(w))) for x in w]
    lens[0] = max(1, lens[0] + total - sum(lens))
    return lens


def _spans(c):
    """(first position, tokens) of each sequence that appends."""
    lens = _lengths(c["tokens"], c["seqs"], 0.6 if c["seqs"] < c["tokens"] else 0.0)
    return [(c["ctx"] + (7 * b) % 13 if c["ctx"] else 0, n) for b, n in enumerate(lens)]


def _pages(lens, page, gen, dev):
    """A page table whose sequences hold distinct pages in shuffled order, and the page count."""
    need = [-(-n // page) for n in lens]
    total = sum(need)
    perm = torch.randperm(total + 1, generator=gen, device=dev).to(torch.int32)
    width = max(need)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    counts = torch.tensor(need, device=dev)
    have = torch.arange(width, device=dev)[None, :] < counts[:, None]
    table[have] = perm[:total]
    return table, total + 1


def _kv_tensors(n_pages, c, gen, dev, fill):
    """K and V pages [n_pages, n_kv, page, hd] as views of the layout's own order."""
    shape = (n_pages, c["n_kv"], c["page"], c["hd"]) if c["layout"] == "head" else \
        (n_pages, c["page"], c["n_kv"], c["hd"])
    out = []
    for scale in fill:
        t = torch.empty(shape, dtype=_DT[c["cache"]], device=dev)
        t.normal_(generator=gen)
        t.mul_(scale)
        out.append(t if c["layout"] == "head" else t.transpose(1, 2))
    return out


def _score_scale(hd):
    """q, k ~ N(0, 1): scores of a few units, as behind normalised q and k."""
    return 2.0 / math.sqrt(hd)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    c = case
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    s = {"case": case}
    if c["op"] == "append":
        T, B, hd = c["tokens"], c["seqs"], c["hd"]
        starts, lens = zip(*_spans(c))
        ends = [a + n for a, n in zip(starts, lens)]
        table, n_pages = _pages(ends, c["page"], gen, dev)
        k, v = _kv_tensors(n_pages, c, gen, dev, (1.0, 1.0))
        heads = c["n_heads"] + 2 * c["n_kv"]
        lt = torch.tensor(lens, device=dev)
        seq = torch.repeat_interleave(torch.arange(B, device=dev), lt)
        first = torch.cumsum(lt, 0) - lt
        pos = torch.arange(T, device=dev) - first[seq] + torch.tensor(starts, device=dev)[seq]
        half = c["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float32) / half)
        ang = torch.arange(max(ends), device=dev, dtype=torch.float32)[:, None] * freq[None, :]
        s.update(qkv=randn(T, heads * hd).to(_DT[c["src"]]), table=table, k=k, v=v, pos=pos.to(torch.int32),
                 seq=seq.to(torch.int32), cos=torch.cos(ang), sin=torch.sin(ang), eps=1e-6,
                 q_norm=1.0 + 0.1 * randn(hd) if c["norm"] else None,
                 k_norm=1.0 + 0.1 * randn(hd) if c["norm"] else None)
        if own:
            from slang_b200 import kernels as kern
            s["cache"] = kern.PagedKV(k, v)
    elif c["op"] == "decode":
        lens = _lengths(c["ctx"] * c["seqs"], c["seqs"], c["spread"])
        table, n_pages = _pages(lens, c["page"], gen, dev)
        k, v = _kv_tensors(n_pages, c, gen, dev, (1.0, 1.0))
        s.update(q=randn(c["seqs"], c["n_heads"], c["hd"]).to(_DT[c["cache"]]), k=k, v=v, table=table,
                 pos=torch.tensor(lens, dtype=torch.int32, device=dev) - 1, scale=_score_scale(c["hd"]))
        if own:
            from slang_b200 import kernels as kern
            s["cache"] = kern.PagedKV(k, v)
            s["workspace"] = kern.attn_decode_paged_workspace(s["cache"], c["n_heads"], c["seqs"])
    elif c["op"] == "prefill":
        lens = _lengths(c["tokens"], c["seqs"], c["spread"])
        T, hd, dt = sum(lens), c["hd"], _DT[c["dtype"]]
        s.update(q=randn(T, c["n_heads"], hd).to(dt), k=randn(T, c["n_kv"], hd).to(dt),
                 v=randn(T, c["n_kv"], hd).to(dt), lens=lens, scale=_score_scale(hd))
        lt = torch.tensor(lens, device=dev)
        s["seq"] = torch.repeat_interleave(torch.arange(len(lens), device=dev), lt)
        s["pos"] = torch.arange(T, device=dev) - (torch.cumsum(lt, 0) - lt)[s["seq"]]
        if own:
            from slang_b200 import kernels as kern
            s["plan"] = kern.PackedPlan(lens, c["n_heads"], c["n_kv"], hd, window=c["window"], device=dev)
    else:
        B, V = c["rows"], c["vocab"]
        x = randn(B, V) * 2.5
        # a few dozen likely tokens stand out of the bulk, as behind a trained head
        hot = torch.randint(0, V, (B, 24), generator=gen, device=dev)
        x.scatter_add_(1, hot, 6.0 + 6.0 * torch.rand(B, 24, generator=gen, device=dev))
        ban = torch.randint(0, V, (B, 64), generator=gen, device=dev)
        x[::4] = x[::4].scatter(1, ban[::4], -math.inf)  # every fourth request bans some tokens
        u = torch.rand(4, B, generator=gen, device=dev)
        row = torch.arange(B, device=dev)
        temp, top_k, top_p, min_p = 0.6 + 0.7 * u[0], torch.zeros(B, device=dev), torch.ones(B, device=dev), \
            torch.zeros(B, device=dev)
        if c["mix"] in ("nucleus", "mixed"):
            top_p = 0.85 + 0.13 * u[1]
        if c["mix"] == "topk":
            top_k = torch.floor(torch.exp(u[2] * math.log(1000.0))).clamp(min=1)
        if c["mix"] == "mixed":  # greedy, nucleus, top-k, min-p, all of them, and plain temperature
            kind = row % 6
            temp = torch.where(kind == 0, torch.zeros_like(temp), temp)
            top_p = torch.where((kind == 2) | (kind == 3) | (kind == 5), torch.ones_like(top_p), top_p)
            top_k = torch.where((kind == 2) | (kind == 4), 20 + torch.floor(180 * u[2]), top_k)
            min_p = torch.where((kind == 3) | (kind == 4), 0.02 + 0.08 * u[3], min_p)
        s.update(logits=x.to(_DT[c["logits"]]), temperature=temp, top_k=top_k.to(torch.int32), top_p=top_p,
                 min_p=min_p, seeds=torch.randint(-2**62, 2**62, (B,), generator=gen, device=dev),
                 pos=torch.randint(0, 100000, (B,), generator=gen, device=dev).to(torch.int32))
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    c = s["case"]
    if own:
        from slang_b200 import kernels as kern
        if c["op"] == "append":
            q = kern.kv_append_paged(s["qkv"], s["cache"], s["table"], s["pos"], s["cos"], s["sin"], c["n_heads"],
                                     seq=s["seq"], q_norm=s["q_norm"], k_norm=s["k_norm"], v_norm=c["norm"],
                                     eps=s["eps"])
            return {"q": q, "k": s["k"], "v": s["v"]}
        if c["op"] == "decode":
            return kern.attn_decode_paged(s["q"], s["cache"], s["table"], s["pos"], scale=s["scale"],
                                          window=c["window"], workspace=s["workspace"])
        if c["op"] == "prefill":
            return kern.attn_prefill_packed(s["q"], s["k"], s["v"], s["plan"], scale=s["scale"])
        return kern.sample(s["logits"], s["seeds"], s["pos"], temperature=s["temperature"], top_k=s["top_k"],
                           top_p=s["top_p"], min_p=s["min_p"])
    return {"append": _append, "decode": _decode, "prefill": _prefill, "sample": _sample}[c["op"]](s)


def _append(s):
    c = s["case"]
    nh, nkv, hd, half = c["n_heads"], c["n_kv"], c["hd"], c["rot"] // 2
    x = s["qkv"].float().view(-1, nh + 2 * nkv, hd)
    q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
    if c["norm"]:
        unit = x / torch.sqrt((x * x).mean(-1, keepdim=True) + s["eps"])
        q, k, v = unit[:, :nh] * s["q_norm"], unit[:, nh:nh + nkv] * s["k_norm"], unit[:, nh + nkv:]
    pos = s["pos"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    qk = torch.cat([q, k], 1)
    a, b, rest = qk[..., :half], qk[..., half:2 * half], qk[..., 2 * half:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(s["k"].dtype)
    page = s["table"][s["seq"].long(), pos // c["page"]].long()
    s["k"][page, :, pos % c["page"]] = qk[:, nh:]
    s["v"][page, :, pos % c["page"]] = v.to(s["v"].dtype)
    return {"q": qk[:, :nh].contiguous(), "k": s["k"], "v": s["v"]}


def _softmax_out(scores, seen, v):
    """softmax over the last axis of the scores that are seen, times v; rows that see nothing give 0."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))


def _decode(s):
    c = s["case"]
    B, nkv, hd = c["seqs"], c["n_kv"], c["hd"]
    pages = s["table"].long().clamp(min=0)
    k = s["k"][pages].transpose(1, 2).reshape(B, nkv, -1, hd).float()
    v = s["v"][pages].transpose(1, 2).reshape(B, nkv, -1, hd).float()
    q = s["q"].float().view(B, nkv, -1, hd)
    scores = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    at, pos = torch.arange(k.shape[2], device=k.device)[None, :], s["pos"].long()[:, None]
    seen = at <= pos
    if c["window"]:
        seen &= at > pos - c["window"]
    out = _softmax_out(scores, seen[:, None, None, :], v)
    return out.reshape(B, c["n_heads"], hd).to(s["q"].dtype)


def _prefill(s):
    c = s["case"]
    nh, nkv, hd = c["n_heads"], c["n_kv"], c["hd"]
    B, L, group = len(s["lens"]), max(s["lens"]), nh // nkv
    seq, pos = s["seq"], s["pos"]

    def padded(x):
        y = torch.zeros(B, L, x.shape[1], hd, dtype=torch.float32, device=x.device)
        y[seq, pos] = x.float()
        return y.transpose(1, 2)

    q, k, v = padded(s["q"]).reshape(B, nkv, group, L, hd), padded(s["k"])[:, :, None], padded(s["v"])[:, :, None]
    scores = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    at = torch.arange(L, device=q.device)
    seen = at[None, :] <= at[:, None]
    if c["window"]:
        seen &= at[None, :] > at[:, None] - c["window"]
    out = _softmax_out(scores, seen, v).view(B, nh, L, hd).transpose(1, 2)
    return out[seq, pos].to(s["q"].dtype)


def _random_words(seeds, pos, n):
    """Philox4x32-10 (Salmon et al., SC 2011) words [rows, n]: key = the row's seed, counter =
    (index / 4, position, 0, 0), word index % 4."""
    k0, k1 = (seeds & _MASK32)[:, None], ((seeds >> 32) & _MASK32)[:, None]
    c0 = torch.arange(-(-n // 4), device=seeds.device)[None, :].expand(seeds.numel(), -1)
    c1 = (pos.long() & _MASK32)[:, None]
    c2 = c3 = torch.zeros_like(c0)
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _MASK32) ^ c1 ^ k0, b & _MASK32, ((a >> 32) & _MASK32) ^ c3 ^ k1, a & _MASK32
        k0, k1 = (k0 + 0x9E3779B9) & _MASK32, (k1 + 0xBB67AE85) & _MASK32
    return torch.stack([c0, c1, c2, c3], -1).view(seeds.numel(), -1)[:, :n]


def _sample(s):
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    B, V = x.shape
    top = x.amax(1, keepdim=True)
    temp = s["temperature"][:, None]
    z = torch.where(x == top, torch.zeros_like(x), x - top) / torch.where(temp > 0, temp, torch.ones_like(temp))
    w = torch.exp(z)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices  # ties: the lowest index first
    rank = torch.arange(V, device=x.device)[None, :]
    top_k, top_p = s["top_k"][:, None], s["top_p"][:, None]
    keep = (rank < top_k) | (top_k <= 0)
    ws = torch.where(keep, w.gather(1, order), torch.zeros_like(w))
    before = torch.cumsum(ws, 1) - ws
    keep &= (before < top_p * ws.sum(1, keepdim=True)) | (rank == 0) | (top_p >= 1)
    keep &= (ws > 0) & (ws >= s["min_p"][:, None])
    keep |= rank == 0
    keep &= (rank == 0) | (temp > 0)
    kept = torch.zeros_like(keep).scatter(1, order, keep)
    u = (_random_words(s["seeds"], s["pos"], V).float() + 0.5) * 2.0 ** -32
    wait = -torch.log1p(-torch.clamp(u, max=1.0 - 2.0 ** -24))  # exponential waiting times: the first to come is drawn
    time = torch.where(kept, wait / w, torch.full_like(w, math.inf))
    first = time == time.amin(1, keepdim=True)
    token = torch.where(first & kept, rank, torch.full_like(rank, V)).amin(1)
    return torch.where(top[:, 0] == -math.inf, torch.full_like(token, -1), token).to(torch.int32)


# ------------------------------------------------------------------ work and the definition in 64 bits

def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    c = case
    if c["op"] == "append":
        T, hd = c["tokens"], c["hd"]
        width = (c["n_heads"] + 2 * c["n_kv"]) * hd
        rows = width * (_size(c["src"]) + _size(c["cache"])) + 12
        places = len({p for a, n in _spans(c) for p in range(a, a + n)})  # each row of the tables is read once
        return {"bytes": T * rows + places * 4 * c["rot"], "flops": 8 * T * width}
    if c["op"] == "decode":
        lens = _lengths(c["ctx"] * c["seqs"], c["seqs"], c["spread"])
        keys = sum(min(n, c["window"]) if c["window"] else n for n in lens)
        return {"bytes": keys * c["n_kv"] * c["hd"] * 4 + c["seqs"] * c["n_heads"] * c["hd"] * 4 + 4 * keys // c["page"],
                "flops": 4 * keys * c["n_heads"] * c["hd"]}
    if c["op"] == "prefill":
        lens = _lengths(c["tokens"], c["seqs"], c["spread"])
        win = c["window"] or 1 << 30
        pairs = sum(n * (n + 1) // 2 if n <= win else win * (win + 1) // 2 + (n - win) * win for n in lens)
        return {"bytes": sum(lens) * (2 * c["n_heads"] + 2 * c["n_kv"]) * c["hd"] * 2,
                "flops": 4 * pairs * c["n_heads"] * c["hd"]}
    return {"bytes": c["rows"] * (c["vocab"] * _size(c["logits"]) + 36), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "append":
        return _append64(s)
    if c["op"] == "decode":
        return _decode64(s)
    if c["op"] == "prefill":
        return _prefill64(s)
    return _sample64(s)


def _append64(s):
    c = s["case"]
    nh, nkv, hd, half = c["n_heads"], c["n_kv"], c["hd"], c["rot"] // 2
    x = s["qkv"].double().view(-1, nh + 2 * nkv, hd)
    pos, seq = s["pos"].long(), s["seq"].long()
    out = torch.empty_like(x)
    for h in range(nh + 2 * nkv):
        y = x[:, h].clone()
        if c["norm"]:
            y = y * (y.square().sum(1, keepdim=True) / hd + s["eps"]).pow(-0.5)
            if h < nh + nkv:
                y = y * (s["q_norm"] if h < nh else s["k_norm"]).double()
        if h < nh + nkv:
            turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())
            pair = torch.complex(y[:, :half], y[:, half:2 * half]) * turn
            y[:, :half], y[:, half:2 * half] = pair.real, pair.imag
        out[:, h] = y
    k, v = s["k"].double().contiguous(), s["v"].double().contiguous()
    page, at = s["table"].long()[seq, pos.div(c["page"], rounding_mode="floor")], pos.remainder(c["page"])
    for g in range(nkv):
        k[page, g, at] = out[:, nh + g]
        v[page, g, at] = out[:, nh + nkv + g]
    return {"q": out[:, :nh].contiguous(), "k": k, "v": v}


def _decode64(s):
    c = s["case"]
    nkv, hd, group = c["n_kv"], c["hd"], c["n_heads"] // c["n_kv"]
    out = torch.zeros(c["seqs"], c["n_heads"], hd, dtype=torch.float64, device=s["q"].device)
    last = s["pos"].tolist()
    for b in range(c["seqs"]):
        lo = max(0, last[b] + 1 - c["window"]) if c["window"] else 0
        at = torch.arange(lo, last[b] + 1, device=out.device)
        page, off = s["table"][b].long()[at // c["page"]], at % c["page"]
        for g in range(nkv):
            q = s["q"][b, g * group:(g + 1) * group].double()
            p = torch.softmax(s["scale"] * q @ s["k"][page, g, off].double().T, -1)
            out[b, g * group:(g + 1) * group] = p @ s["v"][page, g, off].double()
    return out


def _prefill64(s):
    c = s["case"]
    group = c["n_heads"] // c["n_kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    first = 0
    for n in s["lens"]:
        for h in range(c["n_heads"]):
            k = s["k"][first:first + n, h // group].double()
            v = s["v"][first:first + n, h // group].double()
            for lo in range(0, n, 2048):
                hi = min(n, lo + 2048)
                x = s["scale"] * s["q"][first + lo:first + hi, h].double() @ k[:hi].T
                gap = torch.arange(lo, hi, device=x.device)[:, None] - torch.arange(hi, device=x.device)[None, :]
                x[(gap < 0) | (gap >= (c["window"] or n))] = -math.inf
                out[first + lo:first + hi, h] = torch.softmax(x, -1) @ v[:hi]
        first += n
    return out


def _sample64(s):
    rows = []
    words = _random_words(s["seeds"], s["pos"], s["logits"].shape[1])
    for b in range(s["logits"].shape[0]):
        x = s["logits"][b].double()
        temp, k = float(s["temperature"][b]), int(s["top_k"][b])
        p, floor = float(s["top_p"][b]), float(s["min_p"][b])
        order = torch.argsort(x, descending=True, stable=True)
        if temp <= 0:
            rows.append(int(order[0]))
            continue
        order = order[:k] if k > 0 else order
        w = torch.exp((x[order] - x[order[0]]) / temp)
        n = w.numel()
        if p < 1:
            n = min(n, int((torch.cumsum(w, 0) < p * w.sum()).sum()) + 1)
        n = max(1, min(n, int((w >= floor).sum()), int((w > 0).sum())))
        u = (words[b, order[:n]].double() + 0.5) * 2.0 ** -32
        time = -torch.log1p(-u.clamp(max=1 - 2.0 ** -24)) / w[:n]
        rows.append(int(order[:n][time == time.min()].min()))
    return torch.tensor(rows, dtype=torch.int32)
