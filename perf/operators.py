"""Workloads of the 8-bit key/value cache and its attention, with inputs, plain forms, 64-bit results and costs.

A case is one of three ways a program calls them:

  store   the key and value rows of new tokens are quantized into the cache and read back (prefix reuse checks,
          moving a sequence to another cache): qlin_kv_append, then qlin_kv_read of the same rows.
  attend  the query rows of new tokens over their sequences' cached tokens (qlin_kv_attention): decoding, the
          verification of drafted tokens, chunks of a prompt.
  prefix  the same for a batch whose sequences begin with one shared prefix, which is read once for all of them
          (qlin_kv_attention_prefix).

Sequences are ragged, their pages lie scattered, and a batch may hold idle slots (length zero).
"""
from __future__ import annotations

import math

import torch

own = False

_TORCH = {"f16": torch.float16, "f32": torch.float32}
_BYTES = {"f16": 2, "f32": 4}
SCALE_MIN = 2.0 ** -64


def listed():
    # 32 query heads over 8 key/value heads of 128 are those of the 4096 + 1024 + 1024 columns of a Qwen3-4B qkv row
    geo = {"q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "in": "f16", "out": "f16"}
    return [
        # one decoded token into the cache and back, the smallest call
        {"name": "store_1", "kind": "store", "seqs": 1, "len": 1000, "new": 1, "ragged": False, "idle": 0, **geo},
        # one token of each of 64 sequences
        {"name": "store_64x1", "kind": "store", "seqs": 64, "len": 2048, "new": 1, "ragged": True, "idle": 9, **geo},
        # ragged chunks of five prompts, float32 rows, heads of an odd width, small pages
        {"name": "store_5x300_f32", "kind": "store", "seqs": 5, "len": 700, "new": 300, "ragged": True, "idle": 0,
         "q_heads": 10, "kv_heads": 5, "dim": 84, "page": 16, "in": "f32", "out": "f32"},
        # a prompt of 4096 tokens
        {"name": "store_4096", "kind": "store", "seqs": 1, "len": 4096, "new": 4096, "ragged": False, "idle": 0, **geo},
        # one token decoded in a short conversation: latency
        {"name": "decode_1x300", "kind": "attend", "seqs": 1, "len": 300, "new": 1, "ragged": False, "idle": 0, **geo},
        # one token decoded at the reference's longest context
        {"name": "decode_1x32768", "kind": "attend", "seqs": 1, "len": 32768, "new": 1, "ragged": False, "idle": 0, **geo},
        # a serving step: 64 slots at lengths up to 4096, some idle
        {"name": "decode_64x4096", "kind": "attend", "seqs": 64, "len": 4096, "new": 1, "ragged": True, "idle": 9, **geo},
        # drafted tokens verified: up to four rows a sequence, float32 rows as the reference keeps them, heads of 64
        {"name": "verify_8x4_f32", "kind": "attend", "seqs": 8, "len": 2000, "new": 4, "ragged": True, "idle": 0,
         "q_heads": 24, "kv_heads": 8, "dim": 64, "page": 16, "in": "f32", "out": "f32"},
        # a chunk of 512 tokens at the end of a prompt of 8192
        {"name": "chunk_512_of_8192", "kind": "attend", "seqs": 1, "len": 8192, "new": 512, "ragged": False, "idle": 0, **geo},
        # a whole prompt of 4096 tokens
        {"name": "prompt_4096", "kind": "attend", "seqs": 1, "len": 4096, "new": 4096, "ragged": False, "idle": 0, **geo},
        # 32 conversations behind one long system prompt
        {"name": "prefix_32x8192", "kind": "prefix", "seqs": 32, "len": 8704, "prefix": 8192, "new": 1, "ragged": True,
         "idle": 0, **geo},
        # four samples of one prompt with drafted tokens, float32 rows, heads of 256
        {"name": "prefix_4x1024_f32", "kind": "prefix", "seqs": 4, "len": 1150, "prefix": 1024, "new": 4, "ragged": True,
         "idle": 0, "q_heads": 16, "kv_heads": 4, "dim": 256, "page": 32, "in": "f32", "out": "f32"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "prefix", "prefix"])
    dim = rng.choice([64, 128, 128, 128, 256, rng.randint(1, 256)])
    kv = rng.choice([1, 2, 4, 8, 8, rng.randint(1, 12)])
    group = rng.choice([1, 2, 3, 4, 4, 5, 8])
    while kv * group > 32:
        group -= 1
    t = rng.choice(["f16", "f16", "f32"])
    case = {"kind": kind, "q_heads": kv * group, "kv_heads": kv, "dim": dim, "page": rng.choice([16, 32, 64, 64, 128]),
            "in": t, "out": rng.choice([t, t, t, "f16", "f32"]), "ragged": rng.random() < 0.7}
    if kind == "store":
        case["seqs"] = _log_int(rng, 1, 64)
        case["new"] = _log_int(rng, 1, 4096 // case["seqs"])
        case["len"] = min(4096, case["new"] + _log_int(rng, 1, 1024))
    elif kind == "prefix":
        case["seqs"], case["new"] = rng.randint(2, 32), rng.choice([1, 1, 1, 2, 4])
        case["prefix"] = max(1, _log_int(rng, 128, 8192) // case["page"]) * case["page"]
        case["len"] = case["prefix"] + _log_int(rng, 1, 512)
    elif rng.random() < 0.7:  # decoding, verification
        case["seqs"], case["new"] = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 7])
        case["len"] = _log_int(rng, 1, 65536 // case["seqs"] if case["seqs"] > 2 else 32768)
    else:  # prompts
        case["seqs"], case["new"] = rng.choice([1, 1, 2, 4]), _log_int(rng, 16, 1024)
        case["len"] = case["new"] + _log_int(rng, 1, 3000)
    case["new"] = min(case["new"], case["len"])
    case["idle"] = rng.randint(2, 9) if case["seqs"] > 2 and rng.random() < 0.4 else 0
    return case


def _sequences(case):
    """(length after the new rows, new rows) of every sequence."""
    out = []
    floor = case.get("prefix", 0)
    for i in range(case["seqs"]):
        n, new = case["len"], case["new"]
        if case["ragged"] and i:  # the first keeps the full length
            u = (i * 0.6180339887) % 1.0
            new = 1 + int(u * new) if new > 4 else new
            n = floor + max(1, int((n - floor) * (0.05 + 0.95 * ((i * 0.7548776662) % 1.0))))
            new = min(new, n)
        if case["idle"] and i % case["idle"] == case["idle"] - 1:
            n = new = 0
        out.append((n, new))
    return out


# ---- inputs, from the seed alone ---------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _columns(case):
    return -(-case["len"] // case["page"])


def _table(case, seed):
    """int32 [seqs, columns] page ids, scattered over the cache; the prefix's pages are every sequence's."""
    cols, seqs = _columns(case), case["seqs"]
    shared = case.get("prefix", 0) // case["page"]
    perm = torch.randperm(shared + seqs * (cols - shared), generator=_gen(seed * 10 + 1), device="cuda").to(torch.int32)
    return torch.cat([perm[:shared].expand(seqs, shared), perm[shared:].view(seqs, cols - shared)], 1).contiguous()


def _pages(case):
    shared = case.get("prefix", 0) // case["page"]
    return shared + case["seqs"] * (_columns(case) - shared)


def _history(case, seed):
    """Key and value rows of every slot of the cache, [pages, page, kv_heads, dim]: channels of the keys differ in size
    (a few are large, as in trained models), tokens differ in size."""
    g = _gen(seed * 10 + 2)
    shape = (_pages(case), case["page"], case["kv_heads"], case["dim"])
    k = torch.randn(shape, generator=g, device="cuda")
    k *= torch.where(torch.rand(shape[2:], generator=g, device="cuda") < 0.03, 6.0, 1.0)
    v = torch.randn(shape, generator=g, device="cuda")
    v *= torch.rand(shape[:3] + (1,), generator=g, device="cuda") + 0.25
    t = _TORCH[case["in"]]
    return k.to(t), v.to(t)


def _rows(case, seed):
    """New rows of the qkv projection, [rows, (q_heads + 2 kv_heads) * dim]."""
    rows = sum(n for _, n in _sequences(case))
    x = torch.randn((rows, (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]), generator=_gen(seed * 10 + 3),
                    device="cuda")
    return x.to(_TORCH[case["in"]])


def _split(case, x):
    D, hq, hk = case["dim"], case["q_heads"], case["kv_heads"]
    return x[:, :hq * D], x[:, hq * D:(hq + hk) * D], x[:, (hq + hk) * D:]


def _quantize(x):
    """Codes and scales of the last axis; the rounding in 64 bits, where a half is a half."""
    s = (x.float().abs().amax(-1, keepdim=True) / 127.0).clamp_min(SCALE_MIN)
    y = (x.float() * (1.0 / s)).double()
    return (torch.sign(y) * torch.floor(y.abs() + 0.5)).clamp(-127, 127).to(torch.int8), s.squeeze(-1)


# ---- the program's side -------------------------------------------------------------------


def prepare(case, seed):
    seqs = _sequences(case)
    starts = [0]
    for _, n in seqs:
        starts.append(starts[-1] + n)
    state = {"case": case, "seqs": seqs, "x": _rows(case, seed), "table": _table(case, seed)}
    k, v = _history(case, seed)
    length = torch.tensor([n for n, _ in seqs], dtype=torch.int32, device="cuda")
    start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    if own:
        from open_rknpu2_lm_infer_amd import qlinear as ql
        pages, page, hk, D = k.shape
        cache = ql.KVCache(hk, D, pages, page)
        ws = ql.Workspace(1, 256, 256)
        # the history: every page as a full sequence of its own
        ids = torch.arange(pages, dtype=torch.int32, device="cuda").view(pages, 1)
        full = torch.full((pages,), page, dtype=torch.int32, device="cuda")
        all_rows = torch.arange(pages + 1, dtype=torch.int32, device="cuda") * page
        ql.kv_append(ws, cache, ql.KVBatch(all_rows, full, ids, pages * page, page, page),
                     k.view(pages * page, hk * D), v.view(pages * page, hk * D))
        q, nk, nv = _split(case, state["x"])
        batch = ql.KVBatch(start, length, state["table"], starts[-1], max(n for _, n in seqs), case["len"])
        out = _TORCH[case["out"]]
        state.update(ws=ws, cache=cache, batch=batch, q=q, k=nk, v=nv)
        if case["kind"] == "store":
            state["out"] = [torch.empty((starts[-1], hk * D), dtype=out, device="cuda") for _ in range(2)]
        else:
            state["out"] = [torch.empty((starts[-1], case["q_heads"] * D), dtype=out, device="cuda")]
            if case["kind"] == "prefix":
                state["prefix"] = dict(prefix_tokens=case["prefix"], prefix_pages=state["table"][0, :case["prefix"] // page])
        return state
    # the plain form keeps codes and scales as tensors, and where each new row of the batch goes
    (state["ck"], state["sk"]), (state["cv"], state["sv"]) = _quantize(k), _quantize(v)
    state["length"] = length
    state["new"] = torch.tensor([n for _, n in seqs], dtype=torch.int32, device="cuda")
    at = [(i, t, n - m + t) for i, (n, m) in enumerate(seqs) for t in range(m)]
    state["at"] = torch.tensor(at, dtype=torch.int64, device="cuda").view(-1, 3)
    return state


def run(state):
    case = state["case"]
    if own:
        from open_rknpu2_lm_infer_amd import qlinear as ql
        if case["kind"] == "store":
            ql.kv_append(state["ws"], state["cache"], state["batch"], state["k"], state["v"])
            ql.kv_read(state["ws"], state["cache"], state["batch"], state["out"][0], state["out"][1])
        else:
            ql.kv_attention(state["ws"], state["cache"], state["batch"], state["q"], out=state["out"][0],
                            scale=case["dim"] ** -0.5, **state.get("prefix", {}))
        return state["out"]
    return _plain_store(state) if case["kind"] == "store" else _plain_attend(state)


def _plain_store(state):
    case, at = state["case"], state["at"]
    rows, hk, D, P = at.shape[0], case["kv_heads"], case["dim"], case["page"]
    page = state["table"][at[:, 0], at[:, 2] // P].long()
    out = []
    for x, codes, scales in zip(_split(case, state["x"])[1:], (state["ck"], state["cv"]), (state["sk"], state["sv"])):
        c, s = _quantize(x.reshape(rows, hk, D))
        codes[page, at[:, 2] % P], scales[page, at[:, 2] % P] = c, s
        back = codes[page, at[:, 2] % P].float() * scales[page, at[:, 2] % P][..., None]
        out.append(back.view(rows, hk * D).to(_TORCH[case["out"]]))
    return out


def _plain_attend(state):
    case, at = state["case"], state["at"]
    B, T, hq, hk, D = case["seqs"], case["new"], case["q_heads"], case["kv_heads"], case["dim"]
    G = hq // hk
    pages = state["table"].long()

    def dense(codes, scales):  # [B, kv_heads, tokens, dim]
        x = codes[pages].float() * scales[pages][..., None]
        return x.flatten(1, 2).transpose(1, 2)

    q = torch.zeros((B, T, hq, D), device="cuda")
    q[at[:, 0], at[:, 1]] = _split(case, state["x"])[0].float().reshape(-1, hq, D)
    q = q.view(B, T, hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, hk, G * T, D)
    k = dense(state["ck"], state["sk"])
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (D ** -0.5)
    del k
    last = (state["length"] - state["new"])[:, None] + torch.arange(T, device="cuda")
    unseen = torch.arange(x.shape[-1], device="cuda") > last[:, :, None]
    x = x.view(B, hk, G, T, -1).masked_fill_(unseen[:, None, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    o = torch.matmul(x.view(B, hk, G * T, -1), dense(state["cv"], state["sv"]))
    o = o.view(B, hk, G, T, D) / x.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.permute(0, 3, 1, 2, 4)[at[:, 0], at[:, 1]]
    return [o.reshape(-1, hq * D).to(_TORCH[case["out"]])]


# ---- costs and results ----------------------------------------------------------------------


def work(case):
    seqs, D, hk, hq, P = _sequences(case), case["dim"], case["kv_heads"], case["q_heads"], case["page"]
    rows = sum(m for _, m in seqs)
    token = hk * (2 * D + 8)  # codes and scales of a key and a value
    if case["kind"] == "store":  # rows in, codes and scales out and in again, rows out
        return {"bytes": rows * (2 * hk * D * (_BYTES[case["in"]] + _BYTES[case["out"]]) + 2 * token), "flops": rows * 10 * hk * D}
    shared = case.get("prefix", 0)
    tokens = shared + sum(max(n - shared, 0) for n, _ in seqs)
    flops = sum(4 * hq * D * (m * n - m * (m - 1) // 2) for n, m in seqs)
    return {"bytes": tokens * token + rows * hq * D * (_BYTES[case["in"]] + _BYTES[case["out"]]) + 4 * (tokens // P + 1),
            "flops": flops}


def exact(case, seed):
    table, rows = _table(case, seed).cpu(), _rows(case, seed)
    hk, hq, D, P = case["kv_heads"], case["q_heads"], case["dim"], case["page"]

    def stored(x):  # the definition's codes (a float32 scale, its float32 reciprocal, a float32 product) and scale
        top = x.float().abs().max(-1, keepdim=True).values / 127.0
        s = torch.maximum(top, torch.full_like(top, SCALE_MIN))
        y = torch.reciprocal(s) * x.float()
        y = torch.where(y < 0, torch.ceil(y.double() - 0.5), torch.floor(y.double() + 0.5))
        return y * s.double()

    q, k, v = (t.reshape(rows.shape[0], -1, D) for t in _split(case, rows))
    if case["kind"] == "store":
        return [stored(t).reshape(rows.shape[0], hk * D) for t in (k, v)]
    keys, values = _history(case, seed)
    out, r = torch.zeros((rows.shape[0], hq, D), dtype=torch.float64, device="cuda"), 0
    for i, (n, m) in enumerate(_sequences(case)):
        if m == 0:
            continue
        ids = table[i, :-(-n // P)].long().cuda()
        pos = torch.arange(n - m, n, device="cuda")
        for h in range(hk):
            kh = stored(keys[ids, :, h].reshape(-1, D)[:n])
            vh = stored(values[ids, :, h].reshape(-1, D)[:n])
            for g in range(h * (hq // hk), (h + 1) * (hq // hk)):
                a = (q[r:r + m, g].double() @ kh.t()) / math.sqrt(D)
                a[pos[:, None] < torch.arange(n, device="cuda")[None, :]] = -math.inf
                out[r:r + m, g] = torch.softmax(a, 1) @ vh
        r += m
    return [out.reshape(-1, hq * D)]
