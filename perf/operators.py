"""Serving operators of the device library, timed through its C ABI (include/cmol_hip.h).

Four kinds of case, each a dict of plain values:

- window: one layer's decode attention for n sessions whose tokens see a sliding window of
  their own cache and its first few positions (sinks), `cmolhip_attn_window`.
- prompt: the same attention for n consecutive tokens of one session,
  `cmolhip_attn_window_prompt`.
- shared: one layer's decode attention for n sessions that share a prefix (a system prompt)
  cached once, each with positions of its own behind it, `cmolhip_attn_shared`.
- logits: penalties for repeated tokens, biases, grammar masks and the greedy choice on n rows
  of logits, `cmolhip_logits`.

Head shapes and vocabularies are those of the SmolLM2 / SmolLM3 presets (libcmol_amd/synth.py).
Where `own` is false `run` computes the same in elementary torch operations.
"""
import ctypes as C
import math

import numpy as np
import torch

own = False

# heads, kv heads, d_head of the presets
HEADS = {"3b": (16, 4, 128), "360m": (15, 5, 64), "135m": (9, 3, 64), "small": (8, 2, 64)}


def listed():
    return [
        # one token of one chat on the smallest model over the default (fp32) caches: latency
        {"name": "window_one_f32", "kind": "window", "heads": "135m", "n": 1, "lo": 300, "hi": 300, "max_ctx": 2048,
         "window": 128, "sinks": 4, "f16": False},
        # 16 chats of the 360M shape, early and late in their conversations, an odd window
        {"name": "window_16_f32", "kind": "window", "heads": "360m", "n": 16, "lo": 64, "hi": 2000, "max_ctx": 2048,
         "window": 601, "sinks": 1, "f16": False},
        # 32 long chats of the 3B shape in lock-step over fp16 caches
        {"name": "window_32_f16", "kind": "window", "heads": "3b", "n": 32, "lo": 512, "hi": 16384, "max_ctx": 16384,
         "window": 4096, "sinks": 4, "f16": True},
        # a one-line question behind a short chat
        {"name": "prompt_short_f32", "kind": "prompt", "heads": "135m", "n": 45, "pos": 333, "max_ctx": 2048,
         "window": 256, "sinks": 4, "f16": False},
        # a further turn of a served chat
        {"name": "prompt_turn_f16", "kind": "prompt", "heads": "3b", "n": 700, "pos": 5000, "max_ctx": 8192,
         "window": 2048, "sinks": 16, "f16": True},
        # a document as the first prompt, default caches
        {"name": "prompt_long_f32", "kind": "prompt", "heads": "3b", "n": 4096, "pos": 0, "max_ctx": 8192,
         "window": 2048, "sinks": 4, "f16": False},
        # a few chats behind a short system prompt, default caches
        {"name": "shared_5_f32", "kind": "shared", "heads": "135m", "n": 5, "prefix": 777, "lo": 8, "hi": 250,
         "max_ctx": 1024, "f16": False},
        # a full house of 48 chats behind a page of instructions, default caches
        {"name": "shared_48_f32", "kind": "shared", "heads": "3b", "n": 48, "prefix": 2000, "lo": 16, "hi": 500,
         "max_ctx": 1024, "f16": False},
        # 32 chats behind a long document over fp16 caches
        {"name": "shared_32_f16", "kind": "shared", "heads": "3b", "n": 32, "prefix": 8192, "lo": 64, "hi": 2048,
         "max_ctx": 4096, "f16": True},
        # one chat with the default repeat penalty over its last 64 tokens
        {"name": "logits_one", "kind": "logits", "n": 1, "vocab": 49152, "history": 64, "biases": 0, "masks": 0,
         "repeat": True, "counted": False},
        # eight chats under a grammar, a few biased tokens each
        {"name": "logits_8_grammar", "kind": "logits", "n": 8, "vocab": 128256, "history": 128, "biases": 20, "masks": 3,
         "repeat": True, "counted": False},
        # 32 chats, all penalties over their whole histories, a third of them under grammars
        {"name": "logits_32_all", "kind": "logits", "n": 32, "vocab": 128256, "history": 4000, "biases": 300, "masks": 8,
         "repeat": True, "counted": True},
    ]


def _logu(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    kind = rng.choice(["window", "prompt", "shared", "logits"])
    if kind == "logits":
        return {"kind": kind, "n": _logu(rng, 1, 48), "vocab": _logu(rng, 4096, 130000), "history": rng.choice([0, _logu(rng, 1, 6000)]),
                "biases": rng.choice([0, _logu(rng, 1, 300)]), "masks": rng.choice([0, rng.randint(1, 8)]),
                "repeat": rng.random() < 0.7, "counted": rng.random() < 0.5}
    heads = rng.choice(["3b", "360m", "135m", "small"])
    f16 = rng.random() < 0.5
    if kind == "window":
        hi = _logu(rng, 32, 12000)
        return {"kind": kind, "heads": heads, "n": _logu(rng, 1, 48), "lo": max(1, hi // rng.choice([1, 4, 16])), "hi": hi,
                "max_ctx": hi + rng.randint(0, 500), "window": _logu(rng, 16, 4096), "sinks": rng.choice([0, 1, 4, 64]), "f16": f16}
    if kind == "prompt":
        n, pos = _logu(rng, 2, 2500), rng.choice([0, 0, _logu(rng, 16, 6000)])
        return {"kind": kind, "heads": heads, "n": n, "pos": pos, "max_ctx": n + pos + rng.randint(0, 500),
                "window": _logu(rng, 64, 2048), "sinks": rng.choice([0, 1, 4, 64]), "f16": f16}
    hi = _logu(rng, 16, 1500)
    return {"kind": kind, "heads": heads, "n": _logu(rng, 2, 64), "prefix": _logu(rng, 32, 10000), "lo": max(1, hi // rng.choice([1, 8, 64])),
            "hi": hi, "max_ctx": hi + rng.randint(0, 500), "f16": f16}


# ---- inputs -----------------------------------------------------------------------------

def _lens(c):
    """Own lengths of the n sessions, spread evenly over the logarithm of lo..hi."""
    n = c["n"]
    at = [i / (n - 1) if n > 1 else 1.0 for i in range(n)]
    return [max(c["lo"], min(c["hi"], round(c["lo"] * (c["hi"] / c["lo"]) ** t))) for t in at]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dev = "cuda"
    if c["kind"] == "logits":
        n, V, H, B = c["n"], c["vocab"], c["history"], c["biases"]
        s = {"case": c, "x": 3 * torch.randn(n, V, generator=g, device=dev)}
        if H:   # texts repeat their words: ids crowd towards a few, in every order; ragged rows
            ids = (V * torch.rand(n, H, generator=g, device=dev) ** 4).int().clamp(0, V - 1)
            ids = (ids.long() * 7919 % V).int()
            s["ids"] = ids
            s["len"] = torch.randint(0, H + 1, (n,), generator=g, device=dev, dtype=torch.int32)
            s["len"][0] = H
        if c["repeat"]:
            s["repeat"] = 1 + 0.3 * torch.rand(n, generator=g, device=dev)
        if c["counted"]:
            s["freq"] = 0.2 * torch.rand(n, generator=g, device=dev)
            s["pres"] = 0.5 * torch.rand(n, generator=g, device=dev)
        if B:   # every listed id once a row
            s["bias_ids"] = torch.stack([torch.randperm(V, generator=g, device=dev)[:B] for _ in range(n)]).int()
            s["bias"] = 4 * torch.randn(n, s["bias_ids"].shape[1], generator=g, device=dev)
            s["bias_len"] = torch.randint(0, s["bias_ids"].shape[1] + 1, (n,), generator=g, device=dev, dtype=torch.int32)
        if c["masks"]:   # grammar states: from a few allowed tokens to most of them
            words, m = (V + 31) // 32, c["masks"]
            p = 10 ** (-3.5 * torch.rand(m, 1, generator=g, device=dev))
            bits = torch.rand(m, words * 32, generator=g, device=dev) < p
            w = torch.arange(32, device=dev)
            u = (bits.view(m, words, 32).long() << w).sum(2)
            s["mask"] = torch.where(u >= 2 ** 31, u - 2 ** 32, u).int()
            s["mask_row"] = torch.randint(-2 * m, m, (n,), generator=g, device=dev, dtype=torch.int32).clamp_(min=-1)
            s["mask_row"][0] = 0
        s["out"], s["next"] = torch.empty_like(s["x"]), torch.empty(n, dtype=torch.int32, device=dev)
        return s
    h, kv, dh = HEADS[c["heads"]]
    ty = torch.float16 if c["f16"] else torch.float32
    n = c["n"]

    def cache(rows, ctx):
        t = torch.empty(rows, kv, ctx, dh, device=dev, dtype=ty)
        for i in range(rows):
            t[i] = torch.randn(kv, ctx, dh, generator=g, device=dev)
        return t

    s = {"case": c, "q": torch.randn(n, h * dh, generator=g, device=dev)}
    rows = 1 if c["kind"] == "prompt" else n
    s["k"], s["v"] = cache(rows, c["max_ctx"]), cache(rows, c["max_ctx"])
    if c["kind"] != "prompt":
        order = torch.randperm(n, generator=g, device=dev)
        s["lens"] = torch.tensor(_lens(c), dtype=torch.int32, device=dev)[order]
        # sessions sit in the pool's slots in the order they came
        s["slots"] = torch.randperm(n, generator=g, device=dev).int()
    if c["kind"] == "shared":
        s["pk"], s["pv"] = cache(1, c["prefix"]), cache(1, c["prefix"])
    s["out"] = torch.empty_like(s["q"])
    return s


# ---- the library's calls ----------------------------------------------------------------

_ctx = None
_room = None


def _program(need):
    """The context a program makes its kernel calls on, and its workspace (one stream, one call
    after the other, so one workspace serves them all)."""
    global _ctx, _room
    from libcmol_amd import native
    if _ctx is None:
        _ctx = native.Ctx(0)
    if need and (_room is None or _room.numel() < need):
        torch.cuda.synchronize()
        _room = torch.empty(need, dtype=torch.uint8, device="cuda")
    return _ctx.h, C.c_void_p(_room.data_ptr() if need else None), C.c_size_t(need)


def _call(s):
    """The call of a state: entry point and arguments."""
    from libcmol_amd import native
    lib, c = native.lib(), s["case"]

    def p(t):
        return C.c_void_p(s[t].data_ptr() if t in s else None)

    if c["kind"] == "logits":
        d = native.Logits()
        d.n, d.vocab, d.stride = c["n"], c["vocab"], c["vocab"]
        d.logits, d.out, d.next = p("x"), p("out"), p("next")
        if "ids" in s:
            d.history, d.history_len, d.history_cap = p("ids"), p("len"), s["ids"].shape[1]
        d.repeat, d.frequency, d.presence = p("repeat"), p("freq"), p("pres")
        if "bias" in s:
            d.bias_ids, d.bias, d.bias_len, d.bias_cap = p("bias_ids"), p("bias"), p("bias_len"), s["bias"].shape[1]
        if "mask" in s:
            d.mask, d.mask_row, d.mask_rows = p("mask"), p("mask_row"), c["masks"]
        h, room, size = _program(lib.cmolhip_logits_bytes(c["n"], c["vocab"]))
        return lib.cmolhip_logits, (h, C.byref(d), room, size), d
    heads, kv, dh = HEADS[c["heads"]]
    n, ctx, f16 = c["n"], c["max_ctx"], int(c["f16"])
    if c["kind"] == "window":
        h, room, size = _program(lib.cmolhip_attn_window_bytes(n, heads, kv, dh, ctx, c["window"], c["sinks"]))
        return lib.cmolhip_attn_window, (h, n, p("q"), p("k"), p("v"), p("slots"), 0, p("lens"), heads, kv, dh, ctx, f16,
                                         c["window"], c["sinks"], room, size, p("out")), None
    if c["kind"] == "prompt":
        h, room, size = _program(lib.cmolhip_attn_window_prompt_bytes(n, heads, kv, dh, ctx, c["window"], c["sinks"]))
        return lib.cmolhip_attn_window_prompt, (h, n, c["pos"], p("q"), p("k"), p("v"), heads, kv, dh, ctx, f16, c["window"],
                                                c["sinks"], room, size, p("out")), None
    h, room, size = _program(lib.cmolhip_attn_shared_bytes(n, heads, kv, dh, c["prefix"], ctx))
    return lib.cmolhip_attn_shared, (h, n, p("q"), p("pk"), p("pv"), c["prefix"], c["prefix"], p("k"), p("v"), p("slots"), 0,
                                     p("lens"), heads, kv, dh, ctx, f16, room, size, p("out")), None


def _own(s):
    call = s.get("call")
    if call is None or call[3] is not _room:   # (the workspace has grown: its address is another)
        fn, args, kept = _call(s)
        call = s["call"] = (fn, args, kept, _room)
    rc = call[0](*call[1])
    if rc:
        raise RuntimeError("%s failed: %d" % (s["case"]["kind"], rc))
    return {"logits": s["out"], "next": s["next"]} if s["case"]["kind"] == "logits" else s["out"]


# ---- the same in elementary operations --------------------------------------------------

def _soft(scores, seen, values):
    """Weighted means of values [.., T, d] by the softmax of scores [.., R, T] where seen; 0 where
    nothing is."""
    s = torch.where(seen, scores, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    return (e @ torch.where(seen.any(-2).unsqueeze(-1), values, 0.0)) / e.sum(-1, keepdim=True).clamp(min=1e-38)


def _plain_window(s):
    c = s["case"]
    h, kv, dh = HEADS[c["heads"]]
    n, W, S = c["n"], c["window"], c["sinks"]
    L = s["lens"].long().clamp(max=c["max_ctx"])[:, None]
    T = min(S + W, c["max_ctx"])
    at = torch.arange(T, device="cuda")[None]
    first = torch.minimum(L, torch.tensor(S, device="cuda"))   # sinks seen
    begin = torch.maximum(L - W, first)                        # the window behind them
    t = torch.where(at < first, at, begin + at - first)        # [n][T]: visible positions
    seen = t < L
    row = s["slots"].long()[:, None]
    t = t.clamp(max=c["max_ctx"] - 1)
    k = s["k"][row, :, t].float().permute(0, 2, 1, 3).contiguous()   # [n][kv][T][dh]
    v = s["v"][row, :, t].float().permute(0, 2, 1, 3).contiguous()
    q = s["q"].view(n, kv, h // kv, dh)
    scores = (q @ k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(dh))
    return _soft(scores, seen[:, None, None, :], v).reshape(n, h * dh)


def _plain_prompt(s):
    c = s["case"]
    h, kv, dh = HEADS[c["heads"]]
    n, W, S, pos = c["n"], c["window"], c["sinks"], c["pos"]
    first = max(0, pos + 1 - W)
    sinks = min(S, first)
    t = torch.cat([torch.arange(sinks, device="cuda"), torch.arange(first, pos + n, device="cuda")])
    p = pos + torch.arange(n, device="cuda")[:, None]
    seen = (t <= p) & ((t < S) | (t > p - W))
    k, v = s["k"][0][:, t].float(), s["v"][0][:, t].float()
    q = s["q"].view(n, kv, h // kv, dh).permute(1, 2, 0, 3)     # [kv][G][n][dh]
    scores = (q @ k.transpose(1, 2).contiguous()[:, None]) * (1.0 / math.sqrt(dh))
    return _soft(scores, seen, v[:, None]).permute(2, 0, 1, 3).reshape(n, h * dh)


def _plain_shared(s):
    c = s["case"]
    h, kv, dh = HEADS[c["heads"]]
    n, P, T = c["n"], c["prefix"], c["max_ctx"]
    G = h // kv
    q = s["q"].view(n, kv, G, dh)
    rows = q.transpose(0, 1).reshape(kv, n * G, dh)
    sp = (rows @ s["pk"][0].float().transpose(1, 2).contiguous()).view(kv, n, G, P).transpose(0, 1)
    slots = s["slots"].long()
    k, v = s["k"][slots].float(), s["v"][slots].float()
    sc = torch.cat([sp, q @ k.transpose(2, 3).contiguous()], 3) * (1.0 / math.sqrt(dh))
    at = torch.arange(P + T, device="cuda")
    seen = at < P + s["lens"].long()[:, None]
    sc = torch.where(seen[:, None, None], sc, -math.inf)
    e = torch.exp(sc - sc.amax(3, keepdim=True))
    o = e[..., P:].contiguous() @ torch.where(seen[:, None, P:, None], v, 0.0)
    ep = e[..., :P].transpose(0, 1).reshape(kv, n * G, P)
    o = o + (ep @ s["pv"][0].float()).view(kv, n, G, dh).transpose(0, 1)
    return (o / e.sum(3, keepdim=True)).reshape(n, h * dh)


def _plain_logits(s):
    c = s["case"]
    n, V = c["n"], c["vocab"]
    x = s["x"]
    if "ids" in s:
        valid = torch.arange(s["ids"].shape[1], device="cuda") < s["len"][:, None]
        count = torch.zeros(n, V, device="cuda").scatter_add_(1, s["ids"].long(), valid.float())
        if "repeat" in s:   # (the power of a large count passes 32 bits' range)
            f = s["repeat"].double()[:, None] ** count.double()
            x = torch.where(x > 0, x / f, x * f).float()
        if "freq" in s:
            x = x - (s["freq"][:, None] * count + torch.where(count > 0, s["pres"][:, None], 0.0))
    if "bias" in s:
        valid = torch.arange(s["bias"].shape[1], device="cuda") < s["bias_len"][:, None]
        x = x.scatter_add(1, s["bias_ids"].long(), torch.where(valid, s["bias"], 0.0))
    if "mask" in s:
        at = torch.arange(V, device="cuda")
        allowed = (s["mask"][:, at // 32] >> (at % 32).int()) & 1
        ok = (allowed[s["mask_row"].long().clamp(min=0)] != 0) | (s["mask_row"] < 0)[:, None]
        x = torch.where(ok, x, -math.inf)
    top = x.amax(1, keepdim=True)
    index = torch.arange(V, device="cuda", dtype=torch.int32)
    first = torch.where((x == top) & (top > -math.inf), index, V).amin(1)
    return {"logits": x, "next": torch.where(first == V, -1, first).int()}


def run(state):
    if own:
        return _own(state)
    return {"window": _plain_window, "prompt": _plain_prompt, "shared": _plain_shared, "logits": _plain_logits}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "logits":
        n, V = c["n"], c["vocab"]
        b = 8 * n * V + 4 * n * (c["history"] + 2 * c["biases"]) + c["masks"] * V / 8
        return {"bytes": b, "flops": 4 * n * V}
    h, kv, dh = HEADS[c["heads"]]
    per, io = 2 * kv * dh * (2 if c["f16"] else 4), 8 * c["n"] * h * dh
    if c["kind"] == "window":
        vis = sum(min(L, c["sinks"] + c["window"]) for L in _lens(c))
        return {"bytes": vis * per + io, "flops": 4 * vis * h * dh}
    if c["kind"] == "prompt":
        n, pos, W, S = c["n"], c["pos"], c["window"], c["sinks"]
        p = np.arange(pos, pos + n, dtype=np.float64)
        vis = float(np.minimum(p + 1, W + S).sum())
        first = max(0, pos + 1 - W)
        return {"bytes": (min(S, first) + pos + n - first) * per + io, "flops": 4 * vis * h * dh}
    P, own_ = c["prefix"], sum(_lens(c))
    return {"bytes": (P + own_) * per + io, "flops": 4 * (c["n"] * P + own_) * h * dh}


# ---- the definition in 64 bits ----------------------------------------------------------

def _attend(q, k, v, seen=None):
    """One kv head: queries [r][dh] over k, v [T][dh] in 64 bits."""
    a = q.double() @ k.double().T / math.sqrt(q.shape[1])
    if seen is not None:
        a = a.masked_fill(~seen, -math.inf)
    return a.softmax(1) @ v.double()


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "logits":
        x, V = s["x"].double(), c["vocab"]
        for i in range(c["n"]):
            if "ids" in s:
                ids, cnt = s["ids"][i, : int(s["len"][i])].long().unique(return_counts=True)
                y, cnt = x[i, ids], cnt.double()
                if "repeat" in s:
                    y = y * torch.exp(torch.log(s["repeat"][i].double()) * cnt * torch.where(y > 0, -1.0, 1.0))
                if "freq" in s:
                    y = y - s["freq"][i].double() * cnt - s["pres"][i].double()
                x[i, ids] = y
            if "bias" in s:
                m = int(s["bias_len"][i])
                x[i, s["bias_ids"][i, :m].long()] += s["bias"][i, :m].double()
            if "mask" in s and int(s["mask_row"][i]) >= 0:
                w = s["mask"][int(s["mask_row"][i])].cpu().numpy().view(np.uint8)
                bits = torch.from_numpy(np.unpackbits(w, bitorder="little")[:V].astype(bool)).cuda()
                x[i][~bits] = -math.inf
        return {"logits": x, "next": None}
    h, kv, dh = HEADS[c["heads"]]
    n, G = c["n"], h // kv
    q = s["q"].view(n, kv, G, dh)
    out = torch.empty(n, kv, G, dh, device="cuda", dtype=torch.float64)
    if c["kind"] == "prompt":
        pos, W, S = c["pos"], c["window"], c["sinks"]
        for i in range(0, n, 512):
            m = min(512, n - i)
            t = torch.arange(pos + i + m, device="cuda")
            p = pos + i + torch.arange(m, device="cuda")[:, None]
            seen = (t <= p) & ((t < S) | (p - t < W))
            use = seen.any(0)
            for j in range(h):
                out[i:i + m, j // G, j % G] = _attend(q[i:i + m, j // G, j % G], s["k"][0, j // G, : len(t)][use],
                                                      s["v"][0, j // G, : len(t)][use], seen[:, use])
        return out.view(n, h * dh)
    for i in range(n):
        L, r = int(s["lens"][i]), int(s["slots"][i])
        for j in range(kv):
            k, v = s["k"][r, j, :L], s["v"][r, j, :L]
            if c["kind"] == "window":
                a = min(c["sinks"], L)
                b = max(a, L - c["window"])
                k, v = torch.cat([k[:a], k[b:]]), torch.cat([v[:a], v[b:]])
            else:
                k, v = torch.cat([s["pk"][0, j], k]), torch.cat([s["pv"][0, j], v])
            out[i, j] = _attend(q[i, j], k, v)
    return out.view(n, h * dh)
