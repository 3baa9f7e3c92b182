"""Cases of the operators that a layer needs when a batch of answers shares one prompt, and of the
feed-forward half of that layer:

* ``prefix``  -- decode attention over a prefix that every sequence of the batch shares (held once)
  followed by each sequence's own rows, both read from resident caches (fp16 or int8);
* ``gate_up`` -- the gated feed-forward block's first half: both projections, the activation and
  the product, ``act(x Wg^T + bg) * (x Wu^T + bu)``;
* ``linear``  -- a matrix product with bias, activation and residual, ``act(x W^T + b) + r``.

``own`` False: each operator in its plain form, elementary torch operations in 32 bits, rounded
once to the output's type.  ``own`` True: the calls a user makes of ``brimkern_b200``.
"""
import math

import torch

own = False

DEV = "cuda"
_engine = None


def _eng():
    """The program's one engine (library context) on the current GPU."""
    global _engine
    if _engine is None:
        from brimkern_b200.engine import AttentionEngine
        _engine = AttentionEngine(torch.cuda.current_device())
    return _engine


# ---- the cases ------------------------------------------------------------------------------------
def _prefix(name, heads, dim, batch, prefix, rows, tokens=1, q8=False, softcap=0.0, window=0, scale=0.0):
    return {"name": name, "op": "prefix", "heads": heads[0], "kv_heads": heads[1], "dim": dim, "batch": batch,
            "prefix": prefix, "rows": rows, "tokens": tokens, "q8": q8, "softcap": softcap, "window": window,
            "scale": scale}


def _gate_up(name, rows, k, n, act="silu", bias=False):
    return {"name": name, "op": "gate_up", "rows": rows, "k": k, "n": n, "act": act, "bias": bias}


def _linear(name, rows, k, n, act="none", bias=False, residual=False, out="f32"):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "act": act, "bias": bias,
            "residual": residual, "out": out}


def listed():
    return [
        # A few alternatives to one short prompt on a small model: the launch latency counts.
        _prefix("prefix-small", (14, 2), 64, 4, 512, 64),
        # 64 chats behind one 4096-token system prompt, each a few hundred tokens in.
        _prefix("prefix-chats", (32, 8), 128, 64, 4096, 512),
        # 16 answers to one document, two tokens a step (a draft and its check), int8 caches.
        _prefix("prefix-int8", (32, 8), 128, 16, 4099, 777, tokens=2, q8=True),
        # A windowed layer with softcapped scores: only the end of the prefix is seen.
        _prefix("prefix-window", (8, 4), 256, 32, 8192, 512, softcap=50.0, window=4096, scale=1 / 16),
        # 8 questions about one very long document.
        _prefix("prefix-long", (32, 8), 64, 8, 131001, 256),
        # One token of one chat: the weights are streamed once.
        _gate_up("gate-up-token", 1, 2560, 10240),
        # A decode step of a full batch.
        _gate_up("gate-up-batch", 64, 2560, 10240),
        # A short prompt through a layer with biases; nothing is a multiple of a tile.
        _gate_up("gate-up-odd", 77, 2304, 9215, act="gelu_tanh", bias=True),
        # Prompt processing: the products are large.
        _gate_up("gate-up-prompt", 2048, 2560, 10240),
        # The attention output's projection of one token, added to the residual stream.
        _linear("linear-token", 1, 4096, 2560, residual=True),
        # The first half of an image transformer's feed-forward: 257 patches, bias and activation.
        _linear("linear-patches", 257, 1024, 4096, act="quick_gelu", bias=True, out="f16"),
        # The way back from the feed-forward's width to the residual stream, prompt processing.
        _linear("linear-prompt", 2048, 10240, 2560, residual=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_FLOPS = 2.0 * 2048 * 2560 * 10240  # of one product: the largest listed one
MOST_SCORES = 8 * 32 * 131001           # (query row, prefix key) pairs: the largest listed case
MOST_OWN = 64 * 512 * 8 * 128           # elements of the sequences' own K rows


def draw(rng):
    op = rng.choice(["prefix", "prefix", "gate_up", "linear"])
    if op == "prefix":
        (hq, hkv), dim = rng.choice([((14, 2), 64), ((32, 8), 128), ((8, 4), 256), ((32, 8), 64), ((8, 8), 128)])
        tokens = rng.choice([1, 1, 1, 2, 3, 4])
        batch = _log(rng, 1, 64)
        prefix = min(_log(rng, 16, 131001), max(16, MOST_SCORES // (batch * tokens * hq)))
        rows = min(_log(rng, tokens, 2048), max(tokens, MOST_OWN // (batch * hkv * dim)))
        window = rng.choice([0, 0, 0, max(1, (prefix + rows) // 2), 128])
        c = _prefix("", (hq, hkv), dim, batch, prefix, rows, tokens, rng.random() < 0.4,
                    rng.choice([0.0, 0.0, 50.0]), window)
    else:
        rows, k = _log(rng, 1, 2048), 8 * _log(rng, 32, 1280)
        n = _log(rng, 65, 10240)
        n = max(65, min(n, int(MOST_FLOPS / (2.0 * rows * k))))
        act = rng.choice(["none", "silu", "gelu", "gelu_tanh", "quick_gelu"])
        if op == "gate_up":
            c = _gate_up("", rows, k, n, act if act != "none" else "silu", rng.random() < 0.3)
        else:
            c = _linear("", rows, k, n, act, rng.random() < 0.5, rng.random() < 0.5, rng.choice(["f32", "f16"]))
    del c["name"]
    return c


# ---- what a user's program holds before the call ----------------------------------------------------
def _own_lengths(case, seed):
    """Rows of each sequence's own cache after this step's tokens were appended (ragged)."""
    g = torch.Generator().manual_seed(seed * 7919 + 13)
    lo, hi = case["tokens"], case["rows"]
    lens = torch.randint(lo, hi + 1, (case["batch"],), generator=g).tolist()
    lens[0] = hi
    return lens


def _quantised(x):
    """Symmetric int8 codes with one scale per (row, head)."""
    amax = x.abs().amax(-1)
    scale = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax))
    return torch.round(x / scale.unsqueeze(-1)).clamp(-127, 127).to(torch.int8), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    if case["op"] != "prefix":
        rows, k, n = case["rows"], case["k"], case["n"]
        weight = lambda: (normal(n, k) / math.sqrt(k)).half()  # noqa: E731
        s = {"case": case, "x": normal(rows, k).half(), "w": weight()}
        if case["op"] == "gate_up":
            s["w_up"] = weight()
            s["b"], s["b_up"] = (0.1 * normal(n), 0.1 * normal(n)) if case["bias"] else (None, None)
            out = torch.float16
        else:
            s["b"] = 0.1 * normal(n) if case["bias"] else None
            # The residual stream: the sum of the layers before, larger than one layer's part.
            s["r"] = 4.0 * normal(rows, n) if case["residual"] else None
            out = torch.float32 if case["out"] == "f32" else torch.float16
        s["out"] = torch.empty((rows, n), dtype=out, device=DEV)
        if own:
            s["eng"] = _eng()
        return s

    B, T, P, hkv, D = case["batch"], case["tokens"], case["prefix"], case["kv_heads"], case["dim"]
    lens = _own_lengths(case, seed)
    cap = max(lens)
    s = {"case": case, "past": [P + m - T for m in lens],
         "past_dev": torch.tensor([P + m - T for m in lens], device=DEV),
         "q": normal(B, T, case["heads"], D).half(),
         "out": torch.empty((B, T, case["heads"], D), dtype=torch.float16, device=DEV)}
    pk, pv = normal(P, hkv, D), normal(P, hkv, D)
    ok, ov = normal(B, cap, hkv, D), normal(B, cap, hkv, D)
    if case["q8"]:
        s["pk"], s["pv"], s["ok"], s["ov"] = _quantised(pk), _quantised(pv), _quantised(ok), _quantised(ov)
    else:
        s["pk"], s["pv"], s["ok"], s["ov"] = pk.half(), pv.half(), ok.half(), ov.half()
    if own:
        # The resident caches: one sequence for the prefix, one per chat for its own rows.
        from brimkern_b200.engine import AttnConfig, KvCache
        eng = _eng()
        s["eng"] = eng
        s["prefix"] = KvCache(eng.ctx, 1, 1, hkv, D, P, q8=case["q8"])
        s["cache"] = KvCache(eng.ctx, 1, B, hkv, D, cap, q8=case["q8"])
        if case["q8"]:
            s["prefix"].write_codes(0, 0, 0, s["pk"][0], s["pk"][1], s["pv"][0], s["pv"][1])
            for b in range(B):
                s["cache"].write_codes(0, b, 0, s["ok"][0][b], s["ok"][1][b], s["ov"][0][b], s["ov"][1][b])
        else:
            s["prefix"].write_rows(0, 0, 0, s["pk"].float(), s["pv"].float())
            for b in range(B):
                s["cache"].write_rows(0, b, 0, s["ok"][b].float(), s["ov"][b].float())
        s["cfg"] = AttnConfig(case["heads"], hkv, D, scale=case["scale"] or None, softcap=case["softcap"],
                              window=case["window"], kv_offset=P)
    return s


# ---- one pass -----------------------------------------------------------------------------------------
def _act(x, act):
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * (1.0 / math.sqrt(2.0))))
    if act == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))
    if act == "quick_gelu":
        return x / (1.0 + torch.exp(-1.702 * x))
    return x


def _rows32(t, q8):
    return t[0].float() * t[1].unsqueeze(-1) if q8 else t.float()


def _plain_prefix(s):
    c = s["case"]
    B, T, hq, hkv, D, P = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["prefix"]
    pk, pv, ok, ov = (_rows32(s[n], c["q8"]) for n in ("pk", "pv", "ok", "ov"))
    q = s["q"].float().view(B, T, hkv, hq // hkv, D)
    scores = torch.cat([torch.einsum("bthgd,nhd->bthgn", q, pk), torch.einsum("bthgd,bmhd->bthgm", q, ok)], -1)
    scores = scores * (c["scale"] or 1.0 / math.sqrt(D))
    if c["softcap"]:
        scores = c["softcap"] * torch.tanh(scores / c["softcap"])
    pos = s["past_dev"].view(B, 1, 1) + torch.arange(T, device=DEV).view(1, T, 1)
    key = torch.arange(scores.shape[-1], device=DEV).view(1, 1, -1)
    seen = key <= pos
    if c["window"]:
        seen = seen & (key > pos - c["window"])
    scores = scores.masked_fill(~seen.view(B, T, 1, 1, -1), float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.einsum("bthgn,nhd->bthgd", p[..., :P], pv) + torch.einsum("bthgm,bmhd->bthgd", p[..., P:], ov)
    return o.reshape(B, T, hq, D).half()


def run(s):
    c = s["case"]
    if c["op"] == "prefix":
        if own:
            return s["eng"].decodePrefix(s["prefix"], c["prefix"], s["cache"], 0, s["cfg"], s["q"], s["out"], s["past"])
        return _plain_prefix(s)
    if c["op"] == "gate_up":
        if own:
            return s["eng"].ffnGateUp(s["x"], s["w"], s["w_up"], s["out"], act=c["act"], b_gate=s["b"], b_up=s["b_up"])
        x = s["x"].float()
        gate, up = x @ s["w"].float().t(), x @ s["w_up"].float().t()
        if c["bias"]:
            gate, up = gate + s["b"], up + s["b_up"]
        return (_act(gate, c["act"]) * up).half()
    if own:
        return s["eng"].linear(s["x"], s["w"], s["out"], bias=s["b"], act=c["act"], residual=s["r"])
    y = s["x"].float() @ s["w"].float().t()
    if c["bias"]:
        y = y + s["b"]
    y = _act(y, c["act"])
    if c["residual"]:
        y = y + s["r"]
    return y.to(s["out"].dtype)


# ---- what a pass cannot do without --------------------------------------------------------------------
def work(case):
    if case["op"] == "prefix":
        B, T, hq, hkv, D, P = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "dim", "prefix"))
        own_rows = B * (case["rows"] + T) / 2  # ragged lengths, about half of the longest on average
        seen = P
        if case["window"]:
            seen = max(0, min(P, case["window"] - int(own_rows / B)))
            own_rows = min(own_rows, B * case["window"])
        row = 2 * hkv * ((D + 4) if case["q8"] else 2 * D)
        pairs = T * hq * (B * seen + own_rows)
        return {"bytes": (seen + own_rows) * row + 4 * B * T * hq * D, "flops": 4.0 * D * pairs}
    rows, k, n = case["rows"], case["k"], case["n"]
    mats = 2 if case["op"] == "gate_up" else 1
    moved = 2 * rows * k + 2 * mats * n * k + 4 * n * mats * case["bias"]
    if case["op"] == "gate_up":
        moved += 2 * rows * n
    else:
        moved += rows * n * (4 if case["out"] == "f32" else 2) + 4 * rows * n * case["residual"]
    return {"bytes": moved, "flops": 2.0 * mats * rows * k * n}


# ---- the definition in 64 bits ------------------------------------------------------------------------
def _exact_act(x, act):
    if act == "silu":
        return x * torch.special.expit(x)
    if act == "gelu":
        return x * torch.special.ndtr(x)
    if act == "gelu_tanh":
        return x * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3))
    if act == "quick_gelu":
        return x * torch.special.expit(1.702 * x)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] != "prefix":
        out = torch.zeros((case["rows"], case["n"]), dtype=torch.float64, device=DEV)
        x = s["x"].double()
        for j in range(0, case["n"], 1024):  # a block of output columns at a time
            part = slice(j, min(case["n"], j + 1024))
            y = x @ s["w"][part].double().t()
            if s["b"] is not None:
                y = y + s["b"][part].double()
            y = _exact_act(y, case["act"])
            if case["op"] == "gate_up":
                u = x @ s["w_up"][part].double().t()
                if s["b_up"] is not None:
                    u = u + s["b_up"][part].double()
                y = y * u
            elif s["r"] is not None:
                y = y + s["r"][:, part].double()
            out[:, part] = y
        return out
    B, T, hq, hkv, D, P = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "dim", "prefix"))
    G = hq // hkv
    scale = case["scale"] or 1.0 / math.sqrt(D)

    def rows64(t, *at):
        return t[0][at].double() * t[1][at].double().unsqueeze(-1) if case["q8"] else t[at].double()

    out = torch.zeros((B, T, hq, D), dtype=torch.float64, device=DEV)
    pk, pv = rows64(s["pk"], slice(None)), rows64(s["pv"], slice(None))
    for b in range(B):  # one sequence, one token, one kv head at a time: the keys it sees, as one list
        bk, bv = rows64(s["ok"], b), rows64(s["ov"], b)
        for t in range(T):
            end = s["past"][b] + t + 1
            first = max(0, end - case["window"]) if case["window"] else 0
            for h in range(hkv):
                keys = torch.cat([pk[first:min(end, P), h], bk[max(0, first - P):max(0, end - P), h]])
                vals = torch.cat([pv[first:min(end, P), h], bv[max(0, first - P):max(0, end - P), h]])
                z = (s["q"][b, t, h * G:(h + 1) * G].double() @ keys.t()) * scale
                if case["softcap"]:
                    z = torch.tanh(z / case["softcap"]) * case["softcap"]
                out[b, t, h * G:(h + 1) * G] = torch.softmax(z, -1) @ vals
    return out
