"""Cases of further serving operators: the 8-bit paged cache (append, single-token
attention, reading it back), single-token attention for sequences that share a
prefix, and penalties, biases and masks on logits.

`run` computes a case in plain torch operations (32 bits, rounded once at the
end) or, with `own` true, through npu_b200.api. `exact` is the definition in
64 bits, one sequence or row at a time.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
E4M3 = torch.float8_e4m3fn
LARGEST = 448.0  # the largest e4m3 value
SMALLEST_SCALE = 2.0 ** -100  # of a row of zeros (or of values near the smallest floats)


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # One decode step of 64 sequences into an 8-bit cache: every token goes to another sequence's page.
        dict(name="quant_append_step", op="append", batch=64, shortest=1, longest=1, start=5000, hq=32, hkv=4, dim=128,
             page=64, norm=False, rope=128, dtype="bfloat16"),
        # Prompts written to an 8-bit cache after the fused projection, with per-head norms and a partial rotation.
        dict(name="quant_append_prompts", op="append", batch=24, shortest=5, longest=2300, start=37, hq=16, hkv=2,
             dim=256, page=16, norm=True, rope=64, dtype="bfloat16"),
        # One user, a short conversation, small pages (SmolLM2-135M heads, odd group of 3).
        dict(name="quant_decode_one", op="decode", batch=1, shortest=77, longest=77, hq=9, hkv=3, dim=64, page=16,
             gate=False),
        # Gated attention at head dim 256 over long contexts, pages that do not divide a 64-key tile.
        dict(name="quant_decode_gated", op="decode", batch=16, shortest=100, longest=20000, hq=16, hkv=2, dim=256,
             page=48, gate=True),
        # The decode benchmark's sizes with an 8-bit cache: 128 sequences of 1024 to 32768 keys.
        dict(name="quant_decode_many_long", op="decode", batch=128, shortest=1024, longest=32768, hq=32, hkv=4, dim=128,
             page=64, gate=False),
        # The cached part of a few conversations, read back for the attention of their next messages.
        dict(name="gather_chats", op="gather", batch=6, shortest=33, longest=2501, start=0, hkv=3, dim=64, page=16,
             quant=False),
        # Long documents in an 8-bit cache, read back in chunks that start anywhere.
        dict(name="gather_quant_long", op="gather", batch=32, shortest=100, longest=8192, start=500, hkv=4, dim=128,
             page=64, quant=True),
        # A few questions about one short page of instructions: latency.
        dict(name="shared_few", op="shared", batch=3, groups=1, prefix=240, shortest=1, longest=40, hq=9, hkv=3, dim=64,
             page=16, gate=False),
        # Chats behind three different system prompts.
        dict(name="shared_prompts", op="shared", batch=48, groups=3, prefix=2000, shortest=30, longest=1000, hq=9,
             hkv=3, dim=64, page=16, gate=False),
        # Many questions about one long document.
        dict(name="shared_document", op="shared", batch=128, groups=1, prefix=32768, shortest=16, longest=2048, hq=32,
             hkv=4, dim=128, page=64, gate=False),
        # One user's next logits, a conversation of some hundred tokens.
        dict(name="penalize_one", op="penalize", rows=1, vocab=49152, history=300, dtype="float32", bias="none",
             masked=False),
        # A large serving batch: long histories, a bias for all, and a grammar's mask for each row.
        dict(name="penalize_batch", op="penalize", rows=256, vocab=131071, history=4096, dtype="bfloat16", bias="one",
             masked=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "gather", "shared", "shared", "penalize"])
    if op == "penalize":
        vocab = _log(rng, 1000, 131071)
        return dict(op=op, rows=_log(rng, 1, min(256, 33_000_000 // vocab)), vocab=vocab, history=_log(rng, 1, 4096),
                    dtype=rng.choice(["float32", "bfloat16"]), bias=rng.choice(["none", "one", "rows"]),
                    masked=rng.random() < 0.5)
    hq, hkv, dim = rng.choice([(9, 3, 64), (8, 8, 64), (32, 4, 128), (12, 4, 128), (16, 1, 128), (16, 2, 256)])
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "decode":
        longest = _log(rng, 2, 32768)
        batch = _log(rng, 1, max(1, min(128, (128 * 32768 * 4 * 128) // (longest * hkv * dim))))
        return dict(op=op, batch=batch, shortest=_log(rng, 1, longest), longest=longest, hq=hq, hkv=hkv, dim=dim,
                    page=page, gate=rng.random() < 0.3)
    if op == "gather":
        longest = _log(rng, 1, 8192)
        batch = _log(rng, 1, max(1, min(128, (32 * 8192 * 4 * 128) // (longest * hkv * dim))))
        return dict(op=op, batch=batch, shortest=_log(rng, 1, longest), longest=longest,
                    start=rng.choice([0, _log(rng, 1, 6000)]), hkv=hkv, dim=dim, page=page, quant=rng.random() < 0.5)
    if op == "shared":
        prefix = _log(rng, page, 32768) // page * page
        longest = _log(rng, 1, 2048)
        room = (128 * 34816 * 32 * 128) // ((prefix + longest) * max(hq, 8 * hkv) * dim)
        batch = _log(rng, 2, max(2, min(128, room)))
        return dict(op=op, batch=batch, groups=rng.choice([1, 1, _log(rng, 1, batch)]), prefix=prefix,
                    shortest=_log(rng, 1, longest), longest=longest, hq=hq, hkv=hkv, dim=dim, page=page,
                    gate=rng.random() < 0.3)
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


def _groups(case):
    """Offsets of the groups of sequences, and their prefixes: whole pages, the first the longest."""
    batch, groups = case["batch"], min(case["groups"], case["batch"])
    pages = case["prefix"] // case["page"]
    return [batch * g // groups for g in range(groups + 1)], [max(1, pages // (g + 1)) * case["page"] for g in range(groups)]


def work(case):
    if case["op"] == "penalize":
        n, size = case["rows"] * case["vocab"], 4 if case["dtype"] == "float32" else 2
        bias = {"none": 0, "one": 4 * case["vocab"], "rows": 4 * n}[case["bias"]]
        return {"bytes": 2 * n * size + 8 * sum(_histories(case)) + bias + (n // 8 if case["masked"] else 0),
                "flops": 4 * n}
    lens, hkv, dim = _lengths(case), case["hkv"], case["dim"]
    n = sum(lens)
    row = dim + 4  # an 8-bit row with its scale
    if case["op"] == "gather":
        return {"bytes": 2 * n * hkv * (2 * dim + (row if case["quant"] else 2 * dim)), "flops": 2 * n * hkv * dim}
    hq = case["hq"]
    if case["op"] == "decode":
        return {"bytes": 2 * row * n * hkv + 2 * dim * case["batch"] * hq * (3 if case["gate"] else 2) +
                sum(4 * -(-t // case["page"]) for t in lens), "flops": 4 * dim * hq * n}
    if case["op"] == "shared":
        at, prefixes = _groups(case)
        keys = n + sum(prefixes)
        pairs = n + sum((at[g + 1] - at[g]) * p for g, p in enumerate(prefixes))
        return {"bytes": 2 * dim * (2 * keys * hkv + case["batch"] * hq * (3 if case["gate"] else 2)) +
                4 * keys // case["page"], "flops": 4 * dim * hq * pairs}
    size = 4 if case["dtype"] == "float32" else 2
    kept = case["longest"] > 1  # prompts need their rotated keys (and bf16 values) for the attention that follows
    out = 2 * hq + (2 * hkv if kept else 0) + (2 * hkv if kept and size == 4 else 0)
    return {"bytes": n * dim * ((hq + 2 * hkv) * size + out) + 2 * n * hkv * row + n * case["rope"] * size * 2,
            "flops": 6 * n * dim * (hq + hkv)}


# ---------------------------------------------------------------- inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _offsets(lens):
    at = [0]
    for t in lens:
        at.append(at[-1] + t)
    return at


def _histories(case):
    """Tokens so far of each row: up to the case's history, one row without any."""
    rng = random.Random(case["rows"] * 1000003 + case["history"])
    lens = [_log(rng, max(1, case["history"] // 8), case["history"]) for _ in range(case["rows"])]
    lens[0] = case["history"]
    if case["rows"] > 2:
        lens[2] = 0
    return lens


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


def _quantised(x):
    """Rows of x in 8 bits and their scales."""
    scale = (x.abs().amax(-1) / LARGEST).clamp(min=SMALLEST_SCALE)
    return (x / scale[..., None]).clamp(-LARGEST, LARGEST).to(E4M3), scale


def _prepare_penalize(case, gen):
    rows, vocab = case["rows"], case["vocab"]

    def pick(options):
        which = torch.randint(0, len(options), (rows,), generator=gen, device=DEVICE)
        return torch.tensor(options, device=DEVICE)[which]

    lens = _histories(case)
    # Text repeats itself: a few tokens come up often, most once or never.
    tokens = (vocab * torch.rand(rows, max(lens), generator=gen, device=DEVICE) ** 4).long().clamp_(max=vocab - 1)
    tokens = (tokens * 7919) % vocab
    tokens[torch.arange(max(lens), device=DEVICE)[None] >= _ints(lens)[:, None]] = -1
    bias = None
    if case["bias"] != "none":  # a few tokens favoured, some banned
        bias = torch.zeros(rows if case["bias"] == "rows" else 1, vocab, device=DEVICE)
        some = torch.randint(0, vocab, (bias.shape[0], 40), generator=gen, device=DEVICE)
        bias.scatter_(1, some[:, :20], 4 * torch.randn(bias.shape[0], 20, generator=gen, device=DEVICE))
        bias.scatter_(1, some[:, 20:], -math.inf)
        bias = bias if case["bias"] == "rows" else bias[0]
    words = -(-vocab // 32)
    allowed = None
    if case["masked"]:  # a grammar allows anything from a handful to most of the vocabulary
        dense = torch.randint(-2 ** 31, 2 ** 31, (3, rows, words), generator=gen, device=DEVICE, dtype=torch.int64)
        kind = torch.randint(0, 3, (rows, 1), generator=gen, device=DEVICE)
        allowed = torch.where(kind == 0, dense[0] & dense[1] & dense[2], torch.where(kind == 1, dense[0], dense[0] | dense[1]))
        allowed = allowed.to(torch.int32)
    logits = torch.randn(rows, vocab, generator=gen, device=DEVICE) * 2
    return dict(case=case, logits=logits.to(getattr(torch, case["dtype"])), tokens=tokens, lengths=_ints(lens),
                prompt_lengths=_ints([t // 3 for t in lens]), bias=bias, allowed=allowed,
                repetition=pick([1.1, 1.0, 1.3, 0.9] if rows > 1 else [1.1]),
                frequency=pick([0.0, 0.2, -0.1] if rows > 1 else [0.2]),
                presence=pick([0.5, 0.0] if rows > 1 else [0.5]))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device=DEVICE).to(dtype)

    def pools(pages):
        """k and v pages in 8 bits and their scales; rows differ in size."""
        out = {}
        for x in "kv":
            size = 0.2 + 2 * torch.rand(pages, case["hkv"], case["page"], 1, generator=gen, device=DEVICE)
            out[x + "_pages"], out[x + "_scales"] = _quantised(
                size * torch.randn(pages, case["hkv"], case["page"], case["dim"], generator=gen, device=DEVICE))
        return out

    if case["op"] == "penalize":
        return _prepare_penalize(case, gen)
    lens, hkv, dim, page = _lengths(case), case["hkv"], case["dim"], case["page"]
    batch, n = case["batch"], sum(lens)
    if case["op"] == "gather":
        start = [(case["start"] + 7 * b) % (case["start"] + 1) for b in range(batch)]
        table, pages = _paging([s + t for s, t in zip(start, lens)], page, gen)
        st = dict(case=case, table=table, cu=_ints(_offsets(lens)), start=_ints(start), n=n)
        if case["quant"]:
            return {**st, **pools(pages)}
        return dict(st, k_pages=normal(pages, hkv, page, dim), v_pages=normal(pages, hkv, page, dim), k_scales=None,
                    v_scales=None)
    hq = case["hq"]
    if case["op"] == "decode":
        table, pages = _paging(lens, page, gen)
        return dict(case=case, q=normal(batch, hq, dim), table=table, seqlens=_ints(lens),
                    gate=normal(batch, hq, dim) if case["gate"] else None, **pools(pages))
    if case["op"] == "shared":
        at, prefixes = _groups(case)
        own_table, pages = _paging(lens, page, gen)
        counts = [p // page for p in prefixes]
        table = torch.full((batch, max(counts) + own_table.shape[1]), -1, dtype=torch.int32, device=DEVICE)
        for g, c in enumerate(counts):  # the group's pages, then each sequence's own
            rows = slice(at[g], at[g + 1])
            table[rows, :c] = torch.arange(pages, pages + c, dtype=torch.int32, device=DEVICE)
            table[rows, c:c + own_table.shape[1]] = own_table[rows]
            pages += c
        behind = [p for g, p in enumerate(prefixes) for _ in range(at[g], at[g + 1])]
        return dict(case=case, q=normal(batch, hq, dim), k_pages=normal(pages, hkv, page, dim),
                    v_pages=normal(pages, hkv, page, dim), table=table,
                    seqlens=_ints([p + t for p, t in zip(behind, lens)]), prefix_lens=_ints(prefixes),
                    cu_groups=_ints(at) if len(prefixes) > 1 else None,
                    gate=normal(batch, hq, dim) if case["gate"] else None)
    dtype = getattr(torch, case["dtype"])
    start = [(case["start"] + 7 * b) % (case["start"] + 1) for b in range(batch)]
    table, pages = _paging([s + t for s, t in zip(start, lens)], page, gen)
    most = max(s + t for s, t in zip(start, lens))
    inv = 1.0 / (10000.0 ** (torch.arange(0, case["rope"], 2, dtype=torch.float32, device=DEVICE) / case["rope"]))
    angle = torch.outer(torch.arange(most, dtype=torch.float32, device=DEVICE), inv)
    angle = torch.cat([angle, angle], -1)
    qkv = normal(n, (hq + 2 * hkv) * dim, dtype=dtype)  # the fused projection's output; q, k, v are views of it
    return dict(case=case, q=qkv[:, :hq * dim].view(n, hq, dim), k=qkv[:, hq * dim:(hq + hkv) * dim].view(n, hkv, dim),
                v=qkv[:, (hq + hkv) * dim:].view(n, hkv, dim), cos=angle.cos().to(dtype), sin=angle.sin().to(dtype),
                q_norm=(1 + 0.1 * normal(dim, dtype=torch.float32)).to(dtype) if case["norm"] else None,
                k_norm=(1 + 0.1 * normal(dim, dtype=torch.float32)).to(dtype) if case["norm"] else None,
                table=table, cu=_ints(_offsets(lens)), start=_ints(start),
                seqlens=torch.zeros(batch, dtype=torch.int32, device=DEVICE), **pools(pages))


# ---------------------------------------------------------------- plain forms
def _places(st, n):
    """Page and slot of each of n packed tokens, and its position."""
    token = torch.arange(n, device=st["cu"].device)
    which = (token[:, None] >= st["cu"][None, 1:]).sum(1)
    position = token - st["cu"][which] + st["start"][which]
    page = st["case"]["page"]
    return st["table"][which, position // page].long(), position % page, position


def _append(st):
    case = st["case"]
    rope, half = case["rope"], case["rope"] // 2
    page, slot, position = _places(st, st["q"].shape[0])
    cos, sin = st["cos"][position].float()[:, None], st["sin"][position].float()[:, None]

    def rotated(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * w.float()
        turned, rest = x[..., :rope], x[..., rope:]
        turned = turned * cos + torch.cat([-turned[..., half:], turned[..., :half]], -1) * sin
        return torch.cat([turned, rest], -1)

    q, k, v = rotated(st["q"], st["q_norm"]).to(torch.bfloat16), rotated(st["k"], st["k_norm"]), st["v"].float()
    k8, k_scale = _quantised(k)
    v8, v_scale = _quantised(v)
    st["k_pages"].view(torch.uint8)[page, :, slot] = k8.view(torch.uint8)
    st["v_pages"].view(torch.uint8)[page, :, slot] = v8.view(torch.uint8)
    st["k_scales"][page, :, slot] = k_scale
    st["v_scales"][page, :, slot] = v_scale
    st["seqlens"].copy_(st["start"] + st["cu"][1:] - st["cu"][:-1])
    out = {x: st[x] for x in ("k_pages", "v_pages", "k_scales", "v_scales", "seqlens")}
    out["q"] = q
    return {**out, "k": k.to(torch.bfloat16), "v": v.to(torch.bfloat16)} if case["longest"] > 1 else out


def _gather(st):
    page, slot, _ = _places(st, st["n"])

    def read(pages, scales):
        if scales is None:
            return pages[page, :, slot]
        return (pages.view(torch.uint8)[page, :, slot].view(E4M3).float() * scales[page, :, slot][..., None]).to(torch.bfloat16)

    return read(st["k_pages"], st["k_scales"]), read(st["v_pages"], st["v_scales"])


def _softmax_times(s, seen, v):
    """softmax(s over seen) v; s is used up."""
    s.masked_fill_(~seen, -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    return torch.matmul(s, v) / s.sum(-1, keepdim=True)


def _attend(st):
    """One query per sequence over the keys of its table, 8-bit or bf16."""
    case = st["case"]
    q, table = st["q"].float(), st["table"].clamp(min=0).long()
    b, hq, d = q.shape
    at = torch.arange(table.shape[1] * case["page"], device=q.device)
    seen = at[None] < st["seqlens"][:, None]

    def laid_out(pages, scales):
        if scales is None:
            x = pages[table].float()
        else:
            x = pages.view(torch.uint8)[table].view(E4M3).float().mul_(scales[table][..., None])
        return x.transpose(1, 2).reshape(b, case["hkv"], -1, d).masked_fill_(~seen[:, None, :, None], 0)

    s = torch.matmul(q.view(b, case["hkv"], -1, d), laid_out(st["k_pages"], st.get("k_scales")).transpose(-1, -2))
    o = _softmax_times(s.mul_(1 / math.sqrt(d)), seen[:, None, None], laid_out(st["v_pages"], st.get("v_scales")))
    o = o.view(b, hq, d)
    if st["gate"] is not None:
        o = o * torch.sigmoid(st["gate"].float())
    return o.to(torch.bfloat16)


def _penalize(st):
    x = st["logits"].float()
    at = torch.arange(st["tokens"].shape[1], device=x.device)[None]
    there = at < st["lengths"][:, None]
    made = there & (at >= st["prompt_lengths"][:, None])
    tokens = st["tokens"].clamp(min=0)
    seen = torch.zeros_like(x).scatter_add_(1, tokens, there.float()) > 0
    count = torch.zeros_like(x).scatter_add_(1, tokens, made.float())
    r, f, p = st["repetition"][:, None], st["frequency"][:, None], st["presence"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - f * count - p * (count > 0)
    if st["bias"] is not None:
        x = x + st["bias"]
    if st["allowed"] is not None:
        v = torch.arange(x.shape[1], device=x.device)
        x = torch.where((st["allowed"][:, v // 32] >> (v % 32)) & 1 == 1, x, -math.inf)
    return x.to(st["logits"].dtype)


def run(st):
    op = st["case"]["op"]
    if not own:
        return {"append": _append, "decode": _attend, "gather": _gather, "shared": _attend, "penalize": _penalize}[op](st)
    from npu_b200 import api

    if op == "append":
        kept = st["case"]["longest"] > 1
        got = api.rope_append_paged(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["k_pages"], st["v_pages"],
                                    st["table"], st["cu"], start_pos_per_batch=st["start"],
                                    seqlens_out=st["seqlens"], q_norm=st["q_norm"], k_norm=st["k_norm"],
                                    rope_dim=st["case"]["rope"], return_kv=kept, k_scales=st["k_scales"],
                                    v_scales=st["v_scales"])
        out = {x: st[x] for x in ("k_pages", "v_pages", "k_scales", "v_scales", "seqlens")}
        out["q"] = got[0] if kept else got
        return {**out, "k": got[1], "v": got[2]} if kept else out
    if op == "decode":
        return api.decode_paged(st["q"], st["k_pages"], st["v_pages"], st["table"], st["seqlens"],
                                out_dtype=torch.bfloat16, gate=st["gate"], k_scales=st["k_scales"],
                                v_scales=st["v_scales"])
    if op == "gather":
        return api.gather_paged(st["k_pages"], st["v_pages"], st["table"], st["cu"], st["n"],
                                start_pos_per_batch=st["start"], k_scales=st["k_scales"], v_scales=st["v_scales"])
    if op == "shared":
        return api.decode_paged_shared(st["q"], st["k_pages"], st["v_pages"], st["table"], st["seqlens"],
                                       st["prefix_lens"], st["cu_groups"], out_dtype=torch.bfloat16, gate=st["gate"])
    return api.penalize(st["logits"], st["tokens"], st["lengths"], prompt_lengths=st["prompt_lengths"],
                        repetition=st["repetition"], frequency=st["frequency"], presence=st["presence"],
                        bias=st["bias"], allowed=st["allowed"])


# ---------------------------------------------------------------- definitions in 64 bits
def _rows64(pages, scales, ids):
    """All slots of some pages, one after another: [slots, hkv, d]."""
    x = pages[ids] if scales is None else pages.view(torch.uint8)[ids].view(E4M3).double() * scales[ids].double()[..., None]
    return x.double().transpose(1, 2).flatten(0, 1)


def _attend64(st):
    page, parts = st["case"]["page"], []
    for b, t in enumerate(st["seqlens"].tolist()):
        ids = st["table"][b, :-(-t // page)].long()
        k = _rows64(st["k_pages"], st.get("k_scales"), ids)[:t]
        v = _rows64(st["v_pages"], st.get("v_scales"), ids)[:t]
        q = st["q"][b].double().unflatten(0, (k.shape[1], -1))  # [hkv, group, d]
        w = torch.softmax(torch.einsum("hgd,thd->hgt", q, k) / math.sqrt(k.shape[2]), -1)
        parts.append(torch.einsum("hgt,thd->hgd", w, v).flatten(0, 1))
    o = torch.stack(parts)
    return o if st["gate"] is None else o / (1 + torch.exp(-st["gate"].double()))


def _append64(st):
    case = st["case"]
    rope, h, lens, starts, first = case["rope"], case["rope"] // 2, _lengths(case), st["start"].tolist(), 0
    position = torch.cat([torch.arange(s, s + t) for s, t in zip(starts, lens)]).to(DEVICE)

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w.double()
        c, s = st["cos"].double()[position, None], st["sin"].double()[position, None]
        a, b, rest = x[..., :h], x[..., h:rope], x[..., rope:]
        return torch.cat([a * c[..., :h] - b * s[..., :h], b * c[..., h:] + a * s[..., h:], rest], -1)

    q, k, v = turned(st["q"], st["q_norm"]), turned(st["k"], st["k_norm"]), st["v"].double()
    out = {"q": q}
    if case["longest"] > 1:
        out["k"], out["v"] = k, v
    for x, rows in (("k", k), ("v", v)):
        size = torch.linalg.vector_norm(rows, math.inf, -1) / LARGEST
        size = torch.where(size < SMALLEST_SCALE, torch.full_like(size, SMALLEST_SCALE), size)
        out[x + "_pages"], out[x + "_scales"] = st[x + "_pages"].double(), st[x + "_scales"].double()
        first = 0
        for b, (s, t) in enumerate(zip(starts, lens)):
            at = torch.arange(s, s + t, device=DEVICE)
            page, slot = st["table"][b, at // case["page"]].long(), at % case["page"]
            out[x + "_scales"][page, :, slot] = size[first:first + t]
            out[x + "_pages"][page, :, slot] = (rows / size[..., None])[first:first + t]
            first += t
    out["seqlens"] = torch.tensor([s + t for s, t in zip(starts, lens)])
    return out


def _gather64(st):
    case, got = st["case"], []
    for pages, scales in ((st["k_pages"], st["k_scales"]), (st["v_pages"], st["v_scales"])):
        parts = []
        for b, (s, t) in enumerate(zip(st["start"].tolist(), _lengths(case))):
            ids = st["table"][b, :-(-(s + t) // case["page"])].long()
            parts.append(_rows64(pages, scales, ids)[s:s + t])
        got.append(torch.cat(parts))
    return tuple(got)


def _penalize64(st, r):
    x = st["logits"][r].double()
    tokens = st["tokens"][r, :int(st["lengths"][r])]
    made = torch.bincount(tokens[int(st["prompt_lengths"][r]):], minlength=x.shape[0]).double()
    seen = torch.unique(tokens)
    rep = float(st["repetition"][r])
    x[seen] = torch.where(x[seen] < 0, x[seen] * rep, x[seen] / rep)
    x -= float(st["frequency"][r]) * made
    x[made > 0] -= float(st["presence"][r])
    if st["bias"] is not None:
        x += (st["bias"] if st["bias"].dim() == 1 else st["bias"][r]).double()
    if st["allowed"] is not None:
        bits = st["allowed"][r][:, None].bitwise_right_shift(torch.arange(32, device=DEVICE, dtype=torch.int32)) & 1
        x[bits.flatten()[:x.shape[0]] == 0] = -math.inf
    return x


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "penalize":
        return torch.stack([_penalize64(st, r) for r in range(case["rows"])])
    return {"append": _append64, "decode": _attend64, "gather": _gather64, "shared": _attend64}[case["op"]](st)
