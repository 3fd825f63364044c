"""Cases of the serving operators: attention over packed prompts, the paged
key-value cache (append and single-token attention) and token sampling.

`run` computes a case in plain torch operations (32 bits, rounded once at the
end) or, with `own` true, through npu_b200.api. `exact` is the definition in
64 bits, one sequence or row at a time.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # A few one-line prompts arriving together: launch latency.
        dict(name="prompts_short", op="attend", batch=3, shortest=1, longest=40, prefix=0, hq=9, hkv=3, dim=64,
             gate=False),
        # Chat prompts of very different lengths in one packed batch (SmolLM2-135M heads, odd group of 3).
        dict(name="prompts_chat", op="attend", batch=32, shortest=16, longest=2048, prefix=0, hq=9, hkv=3, dim=64,
             gate=False),
        # Long documents, grouped heads 8:1.
        dict(name="prompts_long", op="attend", batch=4, shortest=1024, longest=8192, prefix=0, hq=32, hkv=4, dim=128,
             gate=False),
        # Second chunk of prompts whose first 500 tokens are cached already; gated attention at head dim 256.
        dict(name="prompts_gated_chunk", op="attend", batch=6, shortest=33, longest=2501, prefix=500, hq=16, hkv=2,
             dim=256, gate=True),
        # One user, a short conversation, small pages.
        dict(name="decode_one", op="decode", batch=1, shortest=77, longest=77, hq=9, hkv=3, dim=64, page=16,
             gate=False),
        # A batch of chats in flight, small pages.
        dict(name="decode_chat", op="decode", batch=48, shortest=30, longest=4001, hq=9, hkv=3, dim=64, page=16,
             gate=False),
        # Gated attention at head dim 256 over long contexts, pages that do not divide a 64-key tile.
        dict(name="decode_gated", op="decode", batch=16, shortest=100, longest=20000, hq=16, hkv=2, dim=256, page=48,
             gate=True),
        # The decode benchmark's sizes: 128 sequences of 1024 to 32768 keys.
        dict(name="decode_many_long", op="decode", batch=128, shortest=1024, longest=32768, hq=32, hkv=4, dim=128,
             page=64, gate=False),
        # One decode step of 64 sequences: every token goes to another sequence's page.
        dict(name="append_step", op="append", batch=64, shortest=1, longest=1, start=5000, hq=32, hkv=4, dim=128,
             page=64, norm=False, rope=128, dtype="bfloat16"),
        # Prompts written to the cache after the fused projection, with per-head norms and a partial rotation.
        dict(name="append_prompts", op="append", batch=24, shortest=5, longest=2300, start=37, hq=16, hkv=2, dim=256,
             page=16, norm=True, rope=64, dtype="bfloat16"),
        # One user's next token from float logits.
        dict(name="sample_one", op="sample", rows=1, vocab=49152, dtype="float32"),
        # A large serving batch, each row with its own settings; bf16 logits tie often.
        dict(name="sample_batch", op="sample", rows=256, vocab=131071, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["attend", "decode", "append", "sample"])
    if op == "sample":
        dtype = rng.choice(["float32", "bfloat16"])
        vocab = _log(rng, 1000, 131071)
        return dict(op=op, rows=_log(rng, 1, min(256, 33_000_000 // vocab)), vocab=vocab, dtype=dtype)
    hq, hkv, dim = rng.choice([(9, 3, 64), (8, 8, 64), (32, 4, 128), (12, 4, 128), (16, 1, 128), (16, 2, 256)])
    if op == "attend":
        longest = _log(rng, 2, 8192)
        prefix = rng.choice([0, 0, _log(rng, 1, 1000)])
        room = 4 * 32 * 8192 * 8192 / (hq * longest * (longest + prefix)) * (128 / dim)
        batch = _log(rng, 1, max(1, min(64, int(room))))
        return dict(op=op, batch=batch, shortest=_log(rng, 1, longest), longest=longest, prefix=prefix, hq=hq,
                    hkv=hkv, dim=dim, gate=rng.random() < 0.3)
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "decode":
        longest = _log(rng, 2, 32768)
        batch = _log(rng, 1, max(1, min(128, (128 * 32768 * 4 * 128) // (longest * hkv * dim))))
        return dict(op=op, batch=batch, shortest=_log(rng, 1, longest), longest=longest, hq=hq, hkv=hkv, dim=dim,
                    page=page, gate=rng.random() < 0.3)
    longest = _log(rng, 1, 4000)
    return dict(op=op, batch=_log(rng, 1, max(1, min(256, 24000 // longest))), shortest=_log(rng, 1, longest),
                longest=longest, start=_log(rng, 1, 6000), hq=hq, hkv=hkv, dim=dim, page=page,
                norm=rng.random() < 0.5, rope=rng.choice([dim, dim // 2]), dtype=rng.choice(["float32", "bfloat16"]))


def _lengths(case):
    """Sequence lengths, log-uniform over the case's range, the longest among them: the same for every seed."""
    rng = random.Random(case["batch"] * 1000003 + case["longest"])
    lens = [_log(rng, case["shortest"], case["longest"]) for _ in range(case["batch"])]
    lens[rng.randrange(case["batch"])] = case["longest"]
    return lens


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * ((4 if case["dtype"] == "float32" else 2) + 4) + 8 * case["rows"], "flops": 4 * n}
    lens, hq, hkv, dim = _lengths(case), case["hq"], case["hkv"], case["dim"]
    n = sum(lens)
    if case["op"] == "attend":
        keys = n + case["batch"] * case["prefix"]
        pairs = sum(t * case["prefix"] + t * (t + 1) // 2 for t in lens)
        return {"bytes": 2 * dim * (n * hq * (3 if case["gate"] else 2) + 2 * keys * hkv), "flops": 4 * dim * hq * pairs}
    if case["op"] == "decode":
        return {"bytes": 2 * dim * (2 * n * hkv + case["batch"] * hq * (3 if case["gate"] else 2)) +
                sum(4 * -(-t // case["page"]) for t in lens), "flops": 4 * dim * hq * n}
    size = 4 if case["dtype"] == "float32" else 2
    kept = case["longest"] > 1  # prompts need their rotated keys (and bf16 values) for the attention that follows
    out = hq + 2 * hkv + (hkv if kept else 0) + (hkv if kept and size == 4 else 0)
    return {"bytes": n * dim * ((hq + 2 * hkv) * size + out * 2) + n * case["rope"] * size * 2,
            "flops": 6 * n * dim * (hq + hkv)}


# ---------------------------------------------------------------- inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _offsets(lens):
    at = [0]
    for t in lens:
        at.append(at[-1] + t)
    return at


def _paging(lens, page, gen):
    """A block table over a shuffled pool, with a few pages of other requests in it; unused entries are -1."""
    counts = [-(-t // page) for t in lens]
    width, total = max(counts), sum(counts)
    pages = total + 3
    order = torch.randperm(pages, generator=gen, device=DEVICE)[:total].to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEVICE)
    mask = torch.arange(width, device=DEVICE)[None] < _ints(counts)[:, None]
    table[mask] = order
    return table, pages


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device=DEVICE).to(dtype)

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]

        def pick(options):
            which = torch.randint(0, len(options), (rows,), generator=gen, device=DEVICE)
            return torch.tensor(options, device=DEVICE)[which]

        # Model logits: a broad bulk and a few tokens well above it.
        logits = torch.randn(rows, vocab, generator=gen, device=DEVICE) * 2
        some = torch.randint(0, vocab, (rows, 12), generator=gen, device=DEVICE)
        logits.scatter_add_(1, some, 6 * torch.rand(rows, 12, generator=gen, device=DEVICE) + 2)
        noise = torch.empty(rows, vocab, device=DEVICE).exponential_(generator=gen).clamp_(min=1e-20)
        return dict(case=case, logits=logits.to(getattr(torch, case["dtype"])), noise=noise,
                    temperature=pick([0.7, 1.0, 0.9, 0.0, 1.3] if rows > 1 else [0.8]),
                    top_k=pick([50, 0, 1000, 1, 0, 20] if rows > 1 else [50]).to(torch.int32),
                    top_p=pick([0.9, 1.0, 0.95, 0.5] if rows > 1 else [0.95]),
                    min_p=pick([0.0, 0.0, 0.05] if rows > 1 else [0.0]))
    lens, hq, hkv, dim = _lengths(case), case["hq"], case["hkv"], case["dim"]
    batch, n = case["batch"], sum(lens)
    if case["op"] == "attend":
        klens = [t + case["prefix"] for t in lens]
        keys = sum(klens)
        return dict(case=case, q=normal(n, hq, dim), k=normal(keys, hkv, dim), v=normal(keys, hkv, dim),
                    gate=normal(n, hq, dim) if case["gate"] else None, cu_q=_ints(_offsets(lens)),
                    cu_k=_ints(_offsets(klens)), longest=max(lens), longest_k=max(klens))
    if case["op"] == "decode":
        table, pages = _paging(lens, case["page"], gen)
        return dict(case=case, q=normal(batch, hq, dim), k_pages=normal(pages, hkv, case["page"], dim),
                    v_pages=normal(pages, hkv, case["page"], dim), table=table, seqlens=_ints(lens),
                    gate=normal(batch, hq, dim) if case["gate"] else None)
    dtype = getattr(torch, case["dtype"])
    start = [(case["start"] + 7 * b) % (case["start"] + 1) for b in range(batch)]
    table, pages = _paging([s + t for s, t in zip(start, lens)], case["page"], gen)
    most = max(s + t for s, t in zip(start, lens))
    inv = 1.0 / (10000.0 ** (torch.arange(0, case["rope"], 2, dtype=torch.float32, device=DEVICE) / case["rope"]))
    angle = torch.outer(torch.arange(most, dtype=torch.float32, device=DEVICE), inv)
    angle = torch.cat([angle, angle], -1)
    qkv = normal(n, (hq + 2 * hkv) * dim, dtype=dtype)  # the fused projection's output; q, k, v are views of it
    return dict(case=case, q=qkv[:, :hq * dim].view(n, hq, dim), k=qkv[:, hq * dim:(hq + hkv) * dim].view(n, hkv, dim),
                v=qkv[:, (hq + hkv) * dim:].view(n, hkv, dim), cos=angle.cos().to(dtype), sin=angle.sin().to(dtype),
                q_norm=(1 + 0.1 * normal(dim, dtype=torch.float32)).to(dtype) if case["norm"] else None,
                k_norm=(1 + 0.1 * normal(dim, dtype=torch.float32)).to(dtype) if case["norm"] else None,
                k_pages=normal(pages, hkv, case["page"], dim), v_pages=normal(pages, hkv, case["page"], dim),
                table=table, cu=_ints(_offsets(lens)), start=_ints(start),
                seqlens=torch.zeros(batch, dtype=torch.int32, device=DEVICE))


# ---------------------------------------------------------------- plain forms
def _padded(x, cu, longest):
    """Packed [n, h, d] -> [b, h, longest, d] in 32 bits, and which rows there are."""
    at = torch.arange(longest, device=x.device)
    there = at[None] < (cu[1:] - cu[:-1])[:, None]
    rows = (cu[:-1, None] + at[None]).clamp(max=x.shape[0] - 1)
    y = x[rows.long()].float() * there[:, :, None, None]
    return y.transpose(1, 2), there


def _softmax_times(s, seen, v):
    """softmax(s over seen) v, 0 for rows that see nothing; s is used up."""
    s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = s.sum(-1, keepdim=True)
    return torch.matmul(s, v) / torch.where(total > 0, total, torch.ones_like(total))


def _attend(st):
    case = st["case"]
    group = case["hq"] // case["hkv"]
    q, there = _padded(st["q"], st["cu_q"], st["longest"])
    k, has = _padded(st["k"], st["cu_k"], st["longest_k"])
    v, _ = _padded(st["v"], st["cu_k"], st["longest_k"])
    b, _, lq, d = q.shape
    lens_q, lens_k = st["cu_q"][1:] - st["cu_q"][:-1], st["cu_k"][1:] - st["cu_k"][:-1]
    position = torch.arange(lq, device=q.device)[None] + (lens_k - lens_q)[:, None]
    seen = (torch.arange(k.shape[2], device=q.device)[None, None] <= position[:, :, None]) & has[:, None]
    q = q.reshape(b, case["hkv"], group, lq, d)
    s = torch.matmul(q, k[:, :, None].transpose(-1, -2)).mul_(1 / math.sqrt(d))
    o = _softmax_times(s, seen[:, None, None], v[:, :, None]).reshape(b, -1, lq, d)
    o = o.transpose(1, 2)[there]
    if st["gate"] is not None:
        o = o * torch.sigmoid(st["gate"].float())
    return o.to(torch.bfloat16)


def _decode(st):
    case = st["case"]
    q, table = st["q"].float(), st["table"].clamp(min=0).long()
    b, hq, d = q.shape
    at = torch.arange(table.shape[1] * case["page"], device=q.device)
    seen = at[None] < st["seqlens"][:, None]

    def laid_out(pages):
        x = pages[table].transpose(1, 2).reshape(b, case["hkv"], -1, d).float()
        return x.masked_fill_(~seen[:, None, :, None], 0)

    s = torch.matmul(q.view(b, case["hkv"], -1, d), laid_out(st["k_pages"]).transpose(-1, -2)).mul_(1 / math.sqrt(d))
    o = _softmax_times(s, seen[:, None, None], laid_out(st["v_pages"])).view(b, hq, d)
    if st["gate"] is not None:
        o = o * torch.sigmoid(st["gate"].float())
    return o.to(torch.bfloat16)


def _append(st):
    case = st["case"]
    n, rope, half = st["q"].shape[0], case["rope"], case["rope"] // 2
    token = torch.arange(n, device=st["q"].device)
    which = (token[:, None] >= st["cu"][None, 1:]).sum(1)
    position = token - st["cu"][which] + st["start"][which]
    cos, sin = st["cos"][position].float()[:, None], st["sin"][position].float()[:, None]

    def rotated(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * w.float()
        turned, rest = x[..., :rope], x[..., rope:]
        turned = turned * cos + torch.cat([-turned[..., half:], turned[..., :half]], -1) * sin
        return torch.cat([turned, rest], -1).to(torch.bfloat16)

    q, k, v = rotated(st["q"], st["q_norm"]), rotated(st["k"], st["k_norm"]), st["v"].to(torch.bfloat16)
    page, slot = st["table"][which, position // case["page"]].long(), position % case["page"]
    st["k_pages"][page, :, slot] = k
    st["v_pages"][page, :, slot] = v
    st["seqlens"].copy_(st["start"] + st["cu"][1:] - st["cu"][:-1])
    out = {"q": q, "k_pages": st["k_pages"], "v_pages": st["v_pages"], "seqlens": st["seqlens"]}
    return {**out, "k": k, "v": v} if case["longest"] > 1 else out


def _sample(st):
    x = st["logits"].float()
    temperature = st["temperature"][:, None]
    z = (x - x.amax(-1, keepdim=True)) / torch.where(temperature > 0, temperature, torch.ones_like(temperature))
    w = z.exp()
    ranked, order = torch.sort(x, dim=-1, descending=True, stable=True)  # equal logits: lowest index first
    ws = w.gather(1, order)
    ahead = ws.cumsum(-1) - ws
    k = torch.where(st["top_k"] > 0, st["top_k"], x.shape[1])[:, None]
    p = st["top_p"][:, None]
    keep = (torch.arange(x.shape[1], device=x.device)[None] < k) & (ws >= st["min_p"][:, None])
    keep &= (ahead < p * ws.sum(-1, keepdim=True)) | (p >= 1)
    keep = torch.zeros_like(keep).scatter(1, order, keep)
    drawn = torch.where(keep, w / st["noise"], -1.0).argmax(-1)
    return torch.where(temperature[:, 0] > 0, drawn, x.argmax(-1))


def run(st):
    op = st["case"]["op"]
    if not own:
        return {"attend": _attend, "decode": _decode, "append": _append, "sample": _sample}[op](st)
    from npu_b200 import api

    if op == "attend":
        return api.prefill_varlen(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], out_dtype=torch.bfloat16,
                                  gate=st["gate"])
    if op == "decode":
        return api.decode_paged(st["q"], st["k_pages"], st["v_pages"], st["table"], st["seqlens"],
                                out_dtype=torch.bfloat16, gate=st["gate"])
    if op == "append":
        kept = st["case"]["longest"] > 1
        got = api.rope_append_paged(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["k_pages"], st["v_pages"],
                                    st["table"], st["cu"], start_pos_per_batch=st["start"],
                                    seqlens_out=st["seqlens"], q_norm=st["q_norm"], k_norm=st["k_norm"],
                                    rope_dim=st["case"]["rope"], return_kv=kept)
        out = {"q": got[0] if kept else got, "k_pages": st["k_pages"], "v_pages": st["v_pages"],
               "seqlens": st["seqlens"]}
        return {**out, "k": got[1], "v": got[2]} if kept else out
    return api.sample(st["logits"], st["noise"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                      min_p=st["min_p"])


# ---------------------------------------------------------------- definitions in 64 bits
def _attention64(q, k, v, first):
    """One sequence: q [t, hq, d], k and v [l, hkv, d]; row i sees keys 0 .. first + i."""
    group = q.shape[1] // k.shape[1]
    parts = []
    for h in range(q.shape[1]):
        s = q[:, h].double() @ k[:, h // group].double().T / math.sqrt(q.shape[2])
        late = torch.arange(k.shape[0], device=q.device)[None] > first + torch.arange(q.shape[0], device=q.device)[:, None]
        parts.append(torch.softmax(s.masked_fill(late, -math.inf), -1) @ v[:, h // group].double())
    return torch.stack(parts, 1)


def _sample64(x, e, temperature, top_k, top_p, min_p):
    if temperature == 0:
        return int(x.argmax())
    w, e = torch.exp((x.double() - x.double().max()) / temperature).tolist(), e.double().tolist()
    logits = x.tolist()
    order = sorted(range(len(logits)), key=lambda i: -logits[i])  # stable: equal logits by index
    total, ahead, best, token = math.fsum(w), 0.0, -1.0, -1
    for rank, i in enumerate(order):
        if (top_k > 0 and rank >= top_k) or (top_p < 1 and ahead >= top_p * total) or w[i] < min_p:
            break
        ahead += w[i]
        if w[i] / e[i] > best or (w[i] / e[i] == best and i < token):
            best, token = w[i] / e[i], i
    return token


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        settings = zip(st["temperature"].tolist(), st["top_k"].tolist(), st["top_p"].tolist(), st["min_p"].tolist())
        if case["rows"] * case["vocab"] > 20_000_000:
            return None
        x, e = st["logits"].float().cpu(), st["noise"].cpu()
        return torch.tensor([_sample64(x[r], e[r], *s) for r, s in enumerate(settings)])
    if case["op"] == "attend":
        cu_q, cu_k, parts = st["cu_q"].tolist(), st["cu_k"].tolist(), []
        for b in range(case["batch"]):
            q, k = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
            parts.append(_attention64(st["q"][q], st["k"][k], st["v"][k], case["prefix"]))
        o = torch.cat(parts)
        return o if st["gate"] is None else o / (1 + torch.exp(-st["gate"].double()))
    if case["op"] == "decode":
        parts = []
        for b, t in enumerate(st["seqlens"].tolist()):
            pages = st["table"][b, :-(-t // case["page"])].long()
            k, v = (x[pages].transpose(1, 2).flatten(0, 1)[:t] for x in (st["k_pages"], st["v_pages"]))
            parts.append(_attention64(st["q"][b:b + 1], k, v, t - 1))
        o = torch.cat(parts)
        return o if st["gate"] is None else o / (1 + torch.exp(-st["gate"].double()))
    rope, lens, starts = case["rope"], _lengths(case), st["start"].tolist()
    kp, vp, first = st["k_pages"].double(), st["v_pages"].double(), 0
    position = torch.cat([torch.arange(s, s + t) for s, t in zip(starts, lens)]).to(DEVICE)

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w.double()
        c, s = st["cos"].double()[position, None], st["sin"].double()[position, None]
        a, b, rest = x[..., :rope // 2], x[..., rope // 2:rope], x[..., rope:]
        h = rope // 2
        return torch.cat([a * c[..., :h] - b * s[..., :h], b * c[..., h:] + a * s[..., h:], rest], -1)

    q, k, v = turned(st["q"], st["q_norm"]), turned(st["k"], st["k_norm"]), st["v"].double()
    for b, (s, t) in enumerate(zip(starts, lens)):
        at = torch.arange(s, s + t, device=DEVICE)
        page, slot = st["table"][b, at // case["page"]].long(), at % case["page"]
        kp[page, :, slot], vp[page, :, slot] = k[first:first + t], v[first:first + t]
        first += t
    out = {"q": q, "k_pages": kp, "v_pages": vp, "seqlens": torch.tensor([s + t for s, t in zip(starts, lens)])}
    return {**out, "k": k, "v": v} if case["longest"] > 1 else out
