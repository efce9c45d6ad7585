"""Performance cases of the text path's batch operators: causal attention of packed prompts, and the paged
key/value cache with what fills it and reads it.

The text encoder and text model beside the DiT blocks run batches of requests
of different lengths: prompts packed one after another (a positive and a
negative prompt, the captions of a batch), then new tokens against what is
cached. A step of such a batch is: `paged_plan` (pages and slots from the
requests' lengths), the QKV projection, `qkv_tokens` (head norm, rotation,
query rows, key and value rows into their slots), attention (`prompt_attention`
where the keys are the prompt's own rows, `paged_attention` where they are in
the cache), the output projection. The cases are these four operators.

A case is a dict of plain values; `prepare` makes its inputs on the GPU from
the seed alone, `run` is one pass, `exact` the same result in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _serve():
    """The framework's operators; imported only for its own passes."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-runner_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from llmr_amd import serve
    return serve


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(values):
    return ",".join(str(v) for v in values)


def _ragged(n, lo, hi, key):
    """n lengths spread over [lo, hi] by their logarithm."""
    r = random.Random(key)
    return [max(lo, min(hi, int(round(math.exp(r.uniform(math.log(lo), math.log(hi))))))) for _ in range(n)]


def listed():
    return [
        # the text encoder on one short prompt: latency
        {"name": "prompt_77", "kind": "prompt", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "lens": "77", "pad": 0},
        # a batch of captions of a data set, 24 heads in groups of three, buffers padded to a multiple of 64 rows
        {"name": "prompts_packed_24", "kind": "prompt", "type": "f16", "heads": 24, "kv_heads": 8, "dim": 64,
         "lens": _text(_ragged(24, 12, 512, 5)), "pad": 41},
        # one long prompt: matrix-core bound
        {"name": "prompt_16384", "kind": "prompt", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "lens": "16384", "pad": 0},
        # one request being answered: latency of one token
        {"name": "decode_1", "kind": "paged", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "past": "1100", "new": "1", "pad": 0},
        # a serving batch in its decode phase, ragged contexts, 30 heads in groups of five
        {"name": "decode_64", "kind": "paged", "type": "f16", "heads": 30, "kv_heads": 6, "dim": 128, "page": 16,
         "past": _text(_ragged(64, 100, 12000, 6)), "new": _text([1] * 64), "pad": 0},
        # a few requests with long documents in the cache: HBM bound
        {"name": "decode_long_4", "kind": "paged", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "past": "131000,98304,70001,40000", "new": "1,1,1,1", "pad": 0},
        # a prompt taken in chunks: 512 new tokens behind 30000 cached ones
        {"name": "chunk_512_of_30k", "kind": "paged", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "past": "30001", "new": "512", "pad": 0},
        # chunks and single tokens of many requests in one step, padded to the captured batch's rows
        {"name": "mixed_24", "kind": "paged", "type": "f16", "heads": 16, "kv_heads": 4, "dim": 64, "page": 16,
         "past": _text(_ragged(24, 1, 9000, 7)), "new": _text([1] * 16 + [5, 5, 33, 64, 100, 257, 300, 511]), "pad": 17},
        # the plan of a decode step
        {"name": "plan_decode_32", "kind": "plan", "page": 16, "past": _text(_ragged(32, 1, 4000, 8)),
         "new": _text([1] * 32), "max_pages": 256, "pad": 0},
        # the plan of a step that takes in many prompts
        {"name": "plan_prompts_256", "kind": "plan", "page": 16, "past": _text([0] * 200 + _ragged(56, 1, 3000, 9)),
         "new": _text(_ragged(256, 1, 1000, 10)), "max_pages": 512, "pad": 100},
        # the projection's rows of a decode step, into the cache
        {"name": "qkv_decode_64", "kind": "qkv", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "tokens": 64, "slack": 0, "norm": True, "rope": "halves"},
        # the projection's rows of a long prompt, into the cache
        {"name": "qkv_prompt_8192", "kind": "qkv", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "tokens": 8192, "slack": 100, "norm": True, "rope": "halves"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "paged", "paged", "paged", "plan", "qkv"])
    kv_heads, group = rng.choice([(8, 4), (8, 3), (6, 5), (4, 4), (4, 7), (2, 8), (1, 16), (8, 1), (12, 2)])
    heads = {"type": rng.choice(["bf16", "f16"]), "heads": kv_heads * group, "kv_heads": kv_heads,
             "dim": rng.choice([64, 128, 128])}
    if kind == "prompt":
        total, n = _log(rng, 1, 16384), _log(rng, 1, 64)
        lens = [rng.random() ** 2 + 0.02 for _ in range(n)]
        lens = [int(total * x / sum(lens)) for x in lens]  # short prompts may come out empty
        lens[-1] += total - sum(lens)
        return {"kind": "prompt", **heads, "lens": _text(lens), "pad": rng.choice([0, 0, rng.randint(1, 100)])}
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "paged":
        form = rng.choice(["decode", "chunk", "mixed"])
        n = _log(rng, 1, 128) if form == "decode" else _log(rng, 1, 16)
        if form == "decode":
            new = [rng.choice([1, 1, 1, 2, 4]) if rng.random() < 0.2 else 1 for _ in range(n)]
            past = [_log(rng, 1, min(131072, 300000 // n)) for _ in range(n)]
        else:
            new = [_log(rng, 1, max(1, 2000 // n)) if form == "chunk" or rng.random() < 0.4 else 1 for _ in range(n)]
            past = [rng.choice([0, _log(rng, 1, 32768 // n)]) for _ in range(n)]
        return {"kind": "paged", **heads, "page": page, "past": _text(past), "new": _text(new),
                "pad": rng.choice([0, 0, rng.randint(1, 40)])}
    if kind == "plan":
        n = _log(rng, 1, 512)
        new = [_log(rng, 1, 60000 // n) if rng.random() < 0.7 else rng.randint(0, 1) for _ in range(n)]
        past = [rng.choice([0, _log(rng, 1, 8000)]) for _ in range(n)]
        most = max(-(-(p + m) // page) for p, m in zip(past, new))
        return {"kind": "plan", "page": page, "past": _text(past), "new": _text(new),
                "max_pages": max(1, most) + rng.randint(0, 64), "pad": rng.choice([0, rng.randint(1, 200)])}
    return {"kind": "qkv", **heads, "page": page, "tokens": _log(rng, 1, 8192), "slack": rng.randint(0, 100),
            "norm": rng.random() < 0.5, "rope": rng.choice(["halves", "pairs", "none"])}


# ---- inputs -------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).mul_(std).add_(mean).to(dtype)


def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(lens, page):
    return [-(-n // page) for n in lens]


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case, "kind": case["kind"]}
    if case["kind"] == "plan":
        return _prepare_plan(case, g, s)
    dt = DTYPES[case["type"]]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    s["scale"] = 1.0 / math.sqrt(D)
    if case["kind"] == "qkv":
        return _prepare_qkv(case, g, s, dt)
    # head-normed and rotated queries and keys: about unit size, some heads sharper than others
    new = _ints(case["lens" if case["kind"] == "prompt" else "new"])
    at = _offsets(new)
    T = at[-1] + case["pad"]
    s["at"], s["offsets"] = at, _i32(at)
    s["q"] = _randn(g, T, H, D, std=1.5, dtype=dt)
    s["out"] = torch.zeros(T, H * D, dtype=dt, device=DEV)
    if case["kind"] == "prompt":
        s["k"], s["v"] = (_randn(g, T, Hk, D, dtype=dt) for _ in range(2))
        return s
    page = case["page"]
    kv = [p + n for p, n in zip(_ints(case["past"]), new)]
    need = _pages(kv, page)
    total, most = sum(need), max(need)
    order = torch.randperm(total + 8, generator=g, device=DEV, dtype=torch.int32)  # pages as a used pool hands them out
    table = torch.full((len(kv), most), -1, dtype=torch.int32, device=DEV)
    used = 0
    for i, n in enumerate(need):
        table[i, :n] = order[used:used + n]
        used += n
    s["kv"], s["kv_len"], s["table"], s["page"], s["max_new"] = kv, _i32(kv), table, page, max(new)
    s["k"], s["v"] = (torch.empty(total + 8, Hk, page, D, dtype=dt, device=DEV) for _ in range(2))
    for c in (s["k"], s["v"]):
        for i in range(0, total + 8, 4096):
            c[i:i + 4096] = _randn(g, *c[i:i + 4096].shape, dtype=dt)
    return s


def _prepare_plan(case, g, s):
    page, past, new = case["page"], _ints(case["past"]), _ints(case["new"])
    n = len(past)
    held = _pages(past, page)
    need = [b - a for a, b in zip(held, _pages([p + m for p, m in zip(past, new)], page))]
    order = torch.randperm(sum(held) + sum(need) + 64, generator=g, device=DEV, dtype=torch.int32)
    table = torch.full((n, case["max_pages"]), -1, dtype=torch.int32, device=DEV)
    used = 0
    for i, h in enumerate(held):
        table[i, :h] = order[used:used + h]
        used += h
    s["free"], s["free_count"] = order[used:].contiguous(), _i32([order.numel() - used])
    s["past"], s["new"], s["table"], s["page"] = _i32(past), _i32(new), table, page
    s["tokens"] = sum(new) + case["pad"]
    if own:
        s["batch"] = _serve().PagedBatch.empty(n, s["tokens"], DEV)
    return s


def _prepare_qkv(case, g, s, dt):
    H, Hk, D, T, page = case["heads"], case["kv_heads"], case["dim"], case["tokens"], case["page"]
    n_pages = -(-(T + case["slack"]) // page)
    s["n_heads"], s["n_kv_heads"] = H, Hk
    s["qkv"] = _randn(g, T, (H + 2 * Hk) * D, std=1.7)
    slots = torch.randperm(n_pages * page, generator=g, device=DEV, dtype=torch.int32)[:T]
    if T > 100:  # prompts take whole runs of slots
        slots = torch.sort(slots).values
    s["slots"] = slots.contiguous()
    s["positions"] = torch.randint(0, 16384, (T,), generator=g, device=DEV, dtype=torch.int32)
    s["norms"] = tuple(_randn(g, D, std=0.1, mean=1.0) for _ in range(2)) if case["norm"] else (None, None)
    s["rope"] = None
    if case["rope"] != "none":
        freq = 10000.0 ** (-torch.arange(0, D // 2, dtype=torch.float64, device=DEV) * 2 / D)
        angle = torch.arange(16384, dtype=torch.float64, device=DEV)[:, None] * freq
        s["rope"] = (angle.cos().float(), angle.sin().float())
    s["halves"], s["eps"] = case["rope"] == "halves", 1e-6
    s["q"] = torch.zeros(T, H, D, dtype=dt, device=DEV)
    s["k"], s["v"] = (torch.zeros(n_pages, Hk, page, D, dtype=dt, device=DEV) for _ in range(2))
    return s


# ---- one pass -------------------------------------------------------------------


def run(s):
    kind = s["kind"]
    if own:
        serve = _serve()
        if kind == "prompt":
            return serve.prompt_attention(s["q"], s["k"], s["v"], s["offsets"], s["scale"], out=s["out"])
        if kind == "paged":
            return serve.paged_attention(s["q"], s["k"], s["v"], s["offsets"], s["kv_len"], s["table"], s["max_new"],
                                         s["scale"], out=s["out"])
        if kind == "plan":
            b = serve.paged_plan(s["past"], s["new"], s["free"], s["free_count"], s["table"], s["page"], s["batch"])
            return [b.seq_offsets, b.kv_len, b.slots, b.positions, b.pages, s["table"]]
        serve.qkv_tokens(s["qkv"], s["q"], s["k"], s["v"], slots=s["slots"], positions=s["positions"],
                         q_norm=s["norms"][0], k_norm=s["norms"][1], eps=s["eps"], rope=s["rope"], halves=s["halves"])
        return [s["q"], s["k"], s["v"]]
    return {"prompt": _plain_prompt, "paged": _plain_paged, "plan": _plain_plan, "qkv": _plain_qkv}[kind](s)


def _plain_rows(q, k, v, scale, first, out):
    """Queries q [n, H, D] at positions first .. of keys k, v [Hk, m, D] (f32), each seeing the keys up to its own
    position, into out [n, H * D]."""
    n, H, D = q.shape
    Hk, m = k.shape[0], k.shape[1]
    kt = k.transpose(1, 2).contiguous()
    step = max(1, (1 << 28) // (H * m))
    for a in range(0, n, step):
        b = min(n, a + step)
        seen = min(m, first + b)
        x = q[a:b].float().reshape(b - a, Hk, H // Hk, D).permute(1, 2, 0, 3).reshape(Hk, -1, D)
        p = torch.matmul(x, kt[:, :, :seen].contiguous()).mul_(scale).view(Hk, H // Hk, b - a, seen)
        pos = torch.arange(first + a, first + b, device=DEV)
        p.masked_fill_(torch.arange(seen, device=DEV) > pos[:, None], -math.inf)
        p.sub_(p.amax(dim=-1, keepdim=True)).exp_()
        p.div_(p.sum(dim=-1, keepdim=True))
        o = torch.matmul(p.view(Hk, -1, seen), v[:, :seen]).view(Hk, H // Hk, b - a, D)
        out[a:b] = o.permute(2, 0, 1, 3).reshape(b - a, H * D).to(out.dtype)


def _plain_prompt(s):
    for a, b in zip(s["at"], s["at"][1:]):
        if b > a:
            k, v = (s[x][a:b].float().transpose(0, 1).contiguous() for x in "kv")
            _plain_rows(s["q"][a:b], k, v, s["scale"], 0, s["out"][a:b])
    return s["out"]


def _plain_paged(s):
    page = s["page"]
    for i, (a, b) in enumerate(zip(s["at"], s["at"][1:])):
        if b > a:
            n = s["kv"][i]
            pages = s["table"][i, :-(-n // page)].long()
            k, v = (s[x][pages].transpose(0, 1).reshape(s[x].shape[1], -1, s[x].shape[3])[:, :n].float() for x in "kv")
            _plain_rows(s["q"][a:b], k, v, s["scale"], n - (b - a), s["out"][a:b])
    return s["out"]


def _plain_plan(s):
    past, new, page, table, T = s["past"].long(), s["new"].long(), s["page"], s["table"], s["tokens"]
    n, most = table.shape
    kv = past + new
    offsets = torch.zeros(n + 1, dtype=torch.int64, device=DEV)
    torch.cumsum(new, 0, out=offsets[1:])
    held = (past + page - 1).div(page, rounding_mode="floor")
    want = (kv + page - 1).div(page, rounding_mode="floor") - held
    before = torch.cumsum(want, 0) - want
    col = torch.arange(most, device=DEV)[None]
    taken = (col >= held[:, None]) & (col < (held + want)[:, None])
    rank = before[:, None] + col - held[:, None]
    at = s["free_count"].long() - 1 - rank
    fresh = s["free"][at.clamp(0, s["free"].numel() - 1)]
    table.copy_(torch.where(taken, fresh, table))
    t = torch.arange(T, device=DEV)
    seq = (t[:, None] >= offsets[None, 1:]).sum(dim=1)
    live = seq < n
    seq = seq.clamp(max=n - 1)
    pos = torch.where(live, past[seq] + t - offsets[seq], torch.zeros_like(t))
    slot = table[seq, pos.div(page, rounding_mode="floor")].long() * page + pos % page
    slot = torch.where(live, slot, torch.full_like(slot, -1))
    left = s["free_count"].long() - want.sum()
    pages = torch.cat([left, torch.zeros_like(left)])
    return [offsets.int(), kv.int(), slot.int(), pos.int(), pages.int(), table]


def _plain_norm_rope(x, w, s):
    if w is not None:
        x = x * (1.0 / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + s["eps"])) * w
    if s["rope"] is None:
        return x
    c, sn = (t[s["positions"].long()][:, None] for t in s["rope"])
    D = x.shape[-1]
    a, b = (x[..., :D // 2], x[..., D // 2:]) if s["halves"] else (x[..., 0::2], x[..., 1::2])
    a, b = a * c - b * sn, a * sn + b * c
    return torch.cat([a, b], dim=-1) if s["halves"] else torch.stack([a, b], dim=-1).flatten(-2)


def _plain_qkv(s):
    T, H, D = s["q"].shape
    Hk, page = s["k"].shape[1], s["k"].shape[2]
    x = s["qkv"].view(T, H + 2 * Hk, D)
    s["q"].copy_(_plain_norm_rope(x[:, :H], s["norms"][0], s))
    k, v = _plain_norm_rope(x[:, H:H + Hk], s["norms"][1], s), x[:, H + Hk:]
    at, off = s["slots"].long().div(page, rounding_mode="floor"), s["slots"].long() % page
    s["k"][at, :, off] = k.to(s["k"].dtype)
    s["v"][at, :, off] = v.to(s["v"].dtype)
    return [s["q"], s["k"], s["v"]]


# ---- what a pass cannot do without -------------------------------------------------


def work(case):
    if case["kind"] == "plan":
        past, new, page = _ints(case["past"]), _ints(case["new"]), case["page"]
        T = sum(new) + case["pad"]
        want = sum(b - a for a, b in zip(_pages(past, page), _pages([p + m for p, m in zip(past, new)], page)))
        # lengths in; table entries of half-filled pages and the free list's in; offsets, lengths, slots, positions, entries out
        part = sum(1 for p, m in zip(past, new) if m and p % page)
        return {"bytes": 4 * (2 * len(past) + part + want + 2 * len(past) + 2 * T + want), "flops": 4 * T}
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "qkv":
        T = case["tokens"]
        tables = T * D * 4 if case["rope"] != "none" else 0
        return {"bytes": T * (H + 2 * Hk) * D * 6 + tables + 8 * T, "flops": T * (H + Hk) * D * 6}
    new = _ints(case["lens" if case["kind"] == "prompt" else "new"])
    past = [0] * len(new) if case["kind"] == "prompt" else _ints(case["past"])
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
    kv = sum(p + n for p, n in zip(past, new) if n)
    return {"bytes": 2 * D * (2 * H * sum(new) + 2 * Hk * kv), "flops": 4 * D * H * pairs}


# ---- the result in 64 bits ---------------------------------------------------------


def _exact_rows(q, k, v, scale, first):
    """One key/value head: q [n, G, D], k, v [m, D] -> [n, G, D] in 64 bits; query i sees keys 0 .. first + i."""
    n, G, D = q.shape
    out = torch.empty(n, G, D, dtype=torch.float64, device=DEV)
    k, v = k.double(), v.double()
    step = max(1, (1 << 27) // (G * k.shape[0]))
    for a in range(0, n, step):
        b = min(n, a + step)
        s = torch.tensordot(q[a:b].double(), k, dims=([2], [1])) * scale  # [rows, G, m]
        hidden = torch.arange(k.shape[0], device=DEV)[None, :] > torch.arange(first + a, first + b, device=DEV)[:, None]
        s = torch.where(hidden[:, None, :], torch.full_like(s, -math.inf), s)
        w = torch.exp(s - torch.logsumexp(s, dim=-1, keepdim=True))
        out[a:b] = torch.tensordot(w, v, dims=([2], [0]))
    return out


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    G = H // Hk
    if case["kind"] == "qkv":
        return _exact_qkv(case, s)
    out = s["out"].double()
    for i in range(len(s["at"]) - 1):
        a, b = s["at"][i], s["at"][i + 1]
        if a == b:
            continue
        for h in range(Hk):
            if case["kind"] == "prompt":
                k, v, first = s["k"][a:b, h], s["v"][a:b, h], 0
            else:
                page, n = case["page"], s["kv"][i]
                place = torch.arange(n, device=DEV)
                at = s["table"][i].long()[place // page]
                k, v, first = s["k"][at, h, place % page], s["v"][at, h, place % page], n - (b - a)
            o = _exact_rows(s["q"][a:b, h * G:(h + 1) * G], k, v, s["scale"], first)
            out[a:b, h * G * D:(h + 1) * G * D] = o.reshape(b - a, G * D)
    return out


def _exact_qkv(case, s):
    T, H, D = s["q"].shape
    Hk, page = s["k"].shape[1], s["k"].shape[2]
    x = s["qkv"].double().reshape(T, H + 2 * Hk, D)
    parts = []
    for y, w in ((x[:, :H], s["norms"][0]), (x[:, H:H + Hk], s["norms"][1])):
        if w is not None:
            y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / D + s["eps"]) * w.double()
        if s["rope"] is not None:
            z = torch.complex(*(t.double()[s["positions"].long()] for t in s["rope"]))[:, None, :]
            if s["halves"]:
                y = torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous()) * z
                y = torch.cat([y.real, y.imag], dim=-1)
            else:
                y = torch.view_as_real(torch.view_as_complex(y.reshape(T, -1, D // 2, 2).contiguous()) * z).flatten(-2)
        parts.append(y)
    caches = []
    for c, y in ((s["k"], parts[1]), (s["v"], x[:, H + Hk:])):
        c = c.double().transpose(1, 2).reshape(-1, Hk, D)  # one row a slot
        c[s["slots"].long()] = y
        caches.append(c.view(-1, page, Hk, D).transpose(1, 2).contiguous())
    return [parts[0], caches[0], caches[1]]
