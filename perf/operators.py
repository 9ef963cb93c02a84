"""Operators of 4-bit serving and beam search, over the sizes that the Qwen3 language model's calls and their neighbours
have: products with 4-bit weights, attention over a 4-bit cache, the cache's filling, and a beam search's step.

A value held in 4 bits is s (c - 8): a code c of 0 .. 15 and its group's scale s, an f16 of at most 8 significant bits,
so that the product is exact in f16.
"""
from __future__ import annotations

import math

import torch

own = False

HD = 128        # head width
KV_GROUP = 32   # values of a cache row that share a scale
EOS = 151645    # the token that ends a sequence


def listed() -> list[dict]:
    return [
        # a decode step's q | k | v projection: the smallest call, where latency counts
        {"name": "w4_qkv_m1", "kind": "w4", "m": 1, "k": 2048, "n": 4096, "group": 64, "epi": "plain"},
        # the tied LM head of a decode step: the largest weight that one row reads
        {"name": "w4_head_m1", "kind": "w4", "m": 1, "k": 2048, "n": 151936, "group": 64, "epi": "logits"},
        # gate / up of four beams' step
        {"name": "w4_gateup_m4", "kind": "w4", "m": 4, "k": 2048, "n": 6144, "group": 32, "epi": "swiglu"},
        # down projection of a 10 s clip's prompt, an odd number of rows, added to the residual
        {"name": "w4_down_m409", "kind": "w4", "m": 409, "k": 6144, "n": 2048, "group": 128, "epi": "add"},
        # gate / up of the largest prompt chunk
        {"name": "w4_gateup_m2048", "kind": "w4", "m": 2048, "k": 2048, "n": 6144, "group": 64, "epi": "swiglu"},
        # a decode step after a 10 s clip's prompt, and one over a cache of some hours of speech
        {"name": "attn_t1_p416", "kind": "attn", "b": 1, "t": 1, "p": 417, "qh": 16, "kvh": 8},
        {"name": "attn_t1_p32768", "kind": "attn", "b": 1, "t": 1, "p": 32768, "qh": 16, "kvh": 8},
        # five sequences of different lengths in one step
        {"name": "attn_b5_p3001", "kind": "attn", "b": 5, "t": 1, "p": 3001, "qh": 16, "kvh": 8},
        # the largest prompt chunk over its own rows
        {"name": "attn_t2048", "kind": "attn", "b": 1, "t": 2048, "p": 2048, "qh": 16, "kvh": 8},
        # a prompt's keys and values into the cache, and back as values
        {"name": "fill_t409", "kind": "fill", "b": 1, "t": 409, "kvh": 8},
        # beam search: one step of four beams after a short prompt, of sixteen after a longer one (2 layers' caches)
        {"name": "beam_b4_n448", "kind": "beam", "b": 4, "k": 4, "v": 151936, "n": 448, "p": 512, "layers": 2, "kvh": 8},
        {"name": "beam_b16_n1100", "kind": "beam", "b": 16, "k": 16, "v": 151936, "n": 1100, "p": 1200, "layers": 2,
         "kvh": 8},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
    kind = rng.choice(["w4", "w4", "attn", "attn", "fill", "beam"])
    if kind == "w4":
        epi = rng.choice(["plain", "bias", "add", "swiglu", "logits"])
        m = 1 if rng.random() < 0.3 else _log(rng, 2, 2048)
        k = 8 * _log(rng, 8, 768)
        return {"kind": kind, "m": m, "k": k, "n": _log(rng, 16, 6144 if epi == "swiglu" or m > 64 else 65536),
                "group": rng.choice([32, 64, 128]), "epi": epi}
    if kind == "attn":
        kvh = rng.choice([1, 2, 4, 8])
        qh = kvh * rng.choice([1, 2, 4, 8])
        if rng.random() < 0.6:
            return {"kind": kind, "b": _log(rng, 1, 16), "t": 1, "p": _log(rng, 1, 8192), "qh": qh, "kvh": kvh}
        t = _log(rng, 2, 1024)
        return {"kind": kind, "b": rng.choice([1, 1, 2]), "t": t, "p": t + _log(rng, 1, 1024) - 1, "qh": qh, "kvh": kvh}
    if kind == "fill":
        return {"kind": kind, "b": _log(rng, 1, 4), "t": _log(rng, 1, 2048), "kvh": rng.choice([1, 2, 4, 8])}
    b = _log(rng, 1, 16)
    n = _log(rng, 1, 1024)
    return {"kind": kind, "b": b, "k": b, "v": _log(rng, 500, 151936), "n": n, "p": n + rng.randint(0, 60),
            "layers": rng.randint(1, 2), "kvh": rng.choice([2, 4, 8])}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape) -> torch.Tensor:
    return torch.randn(*shape, device="cuda", generator=g)


def _padded(t: torch.Tensor, group: int) -> torch.Tensor:
    """Rows of zeros up to whole groups along the first axis."""
    extra = -t.shape[0] % group
    return torch.cat([t, t.new_zeros(extra, *t.shape[1:])]) if extra else t


def _scale(amax: torch.Tensor) -> torch.Tensor:
    """f32 > 0 rounded up to 8 significant bits, to a multiple of 2^-24 below 2^-17, at most 8128, as f16."""
    bits = (amax.contiguous().view(torch.int32) + 0xFFFF) & -0x10000
    s = bits.view(torch.float32)
    s = torch.where(s < 2.0 ** -17, torch.ceil(amax * 2.0 ** 24) * 2.0 ** -24, s)
    return s.clamp(max=8128.0).half()


def _quantize(x: torch.Tensor):
    """x f16[..., G] -> codes u8[..., G], scales f16[...]."""
    xf = x.float()
    seven = xf.new_tensor(7.0)  # a division proper: by a number it would be a product with 1 / 7
    s = _scale(torch.maximum(xf.amax(-1).clamp(min=0) / seven, -xf.amin(-1).clamp(max=0) / 8))
    sf = s.float().unsqueeze(-1)
    c = torch.where(sf > 0, torch.floor(xf / sf + 0.5), torch.zeros_like(xf)).clamp(-8, 7)
    return (c + 8).to(torch.uint8), s


def _weight(g, k: int, n: int, group: int):
    """A weight as a checkpoint holds it: codes u8[K, N], scales f16[ceil(K / G), N]."""
    groups = -(-k // group)
    codes = torch.randint(0, 16, (k, n), device="cuda", generator=g, dtype=torch.uint8)
    amax = (0.5 + torch.rand(groups, n, device="cuda", generator=g)) * (0.2 / math.sqrt(k))
    return codes, _scale(amax)


def _cache_rows(g, b: int, kvh: int, p: int):
    """Keys and values f16[B, P, kvh 128] as they come from a projection: heads of their own size."""
    size = torch.exp(0.5 * _randn(g, 1, 1, kvh, 1))
    k = (_randn(g, b, p, kvh, HD) * size).half().reshape(b, p, kvh * HD)
    v = (_randn(g, b, p, kvh, HD) * size).half().reshape(b, p, kvh * HD)
    return k, v


def _inputs(case: dict, seed: int) -> dict:
    g, c = _gen(seed), case
    if c["kind"] == "w4":
        s = {"x": _randn(g, c["m"], c["k"]).half()}
        s["w"] = [_weight(g, c["k"], c["n"], c["group"]) for _ in range(2 if c["epi"] == "swiglu" else 1)]
        s["extra"] = _randn(g, c["n"]).half() if c["epi"] == "bias" else _randn(g, c["m"], c["n"]).half()
        return s
    if c["kind"] == "attn":
        k, v = _cache_rows(g, c["b"], c["kvh"], c["p"])
        # the first sequence fills the cache; the others end anywhere before
        pos = torch.randint(0, c["p"] - c["t"] + 1, (c["b"],), device="cuda", generator=g)
        pos[0] = c["p"] - c["t"]
        return {"k": k, "v": v, "pos": pos, "q": _randn(g, c["b"] * c["t"], c["qh"] * HD).half()}
    if c["kind"] == "fill":
        k, v = _cache_rows(g, c["b"], c["kvh"], c["t"])
        return {"k": k, "v": v, "pos": torch.zeros(c["b"], dtype=torch.int64, device="cuda")}
    rows = [_cache_rows(g, c["b"], c["kvh"], c["p"]) for _ in range(c["layers"])]
    done = (torch.rand(c["b"], device="cuda", generator=g) < 0.15).long()
    done[0] = 0
    return {"rows": rows, "logits": 3 * _randn(g, c["b"], c["v"]), "scores": -5 * torch.rand(c["b"], device="cuda", generator=g),
            "done": done, "n": torch.tensor([c["n"]], device="cuda"), "eos": min(EOS, c["v"] - 1)}


def _rows_q4(k: torch.Tensor, v: torch.Tensor, kvh: int):
    """k, v f16[B, P, kvh 128] -> codes u8[B, 2, kvh, P, 128], scales f16[B, 2, kvh, P, 4]."""
    b, p, _ = k.shape
    x = torch.stack([k, v], 1).view(b, 2, p, kvh, HD // KV_GROUP, KV_GROUP).transpose(2, 3)
    codes, scales = _quantize(x)
    return codes.reshape(b, 2, kvh, p, HD), scales


def _ceil32(p: int) -> int:
    return -(-p // 32) * 32


def prepare(case: dict, seed: int) -> dict:
    s, c = _inputs(case, seed), case
    s["case"] = dict(c)
    if own:
        # what a serving program keeps: the weights laid out once, the caches as earlier calls filled them
        import lokinfer_amd as lk

        q4, T = lk.ops.q4_gpu, lk.Tensor
        s["lk"] = lk
        if c["kind"] == "w4":
            s["w"] = [q4.pack_w4(T(codes), T(scales), c["group"]) for codes, scales in s["w"]]
        elif c["kind"] != "fill":
            layers = [(s.pop("k"), s.pop("v"))] if c["kind"] == "attn" else s.pop("rows")
            kv = torch.zeros(len(layers), c["b"], 2, c["kvh"], 72 * _ceil32(c["p"]), dtype=torch.uint8, device="cuda")
            zero = T(torch.zeros(c["b"], dtype=torch.int64, device="cuda"))
            for i, (k, v) in enumerate(layers):
                q4.kv4_write_f16_gpu(T(kv[i]), T(k.reshape(-1, k.shape[2])), T(v.reshape(-1, v.shape[2])), zero)
            s["kv"] = T(kv[0] if c["kind"] == "attn" else kv)
        else:
            s["kv"] = q4.kv4_cache(c["b"], c["kvh"], c["t"])
            s["k"], s["v"] = (x.view(-1, c["kvh"] * HD) for x in (s["k"], s["v"]))
        for name, x in s.items():
            if isinstance(x, torch.Tensor):
                s[name] = T(x)
    elif c["kind"] == "attn":
        s["codes"], s["scales"] = _rows_q4(s.pop("k"), s.pop("v"), c["kvh"])
    elif c["kind"] == "beam":
        held = [_rows_q4(k, v, c["kvh"]) for k, v in s.pop("rows")]
        s["codes"], s["scales"] = (torch.stack(x) for x in zip(*held))
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------

def _values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """f32 values of codes u8[..., 128] under scales f16[..., 4]."""
    c = codes.view(*codes.shape[:-1], -1, KV_GROUP).float() - 8
    return (c * scales.float().unsqueeze(-1)).flatten(-2)


def _plain_w4(s: dict, c: dict):
    x = s["x"].float()

    def product(w):
        codes, scales = w
        grouped = _padded(codes.float() - 8, c["group"]).view(-1, c["group"], c["n"])
        return x @ (grouped * scales.float().unsqueeze(1)).view(-1, c["n"])[: c["k"]]

    y = product(s["w"][0])
    if c["epi"] == "swiglu":
        y = y / (1 + torch.exp(-y)) * product(s["w"][1])
    elif c["epi"] in ("bias", "add"):
        y = y + s["extra"].float()
    return y if c["epi"] == "logits" else y.half()


def _plain_attn(s: dict, c: dict):
    b, t, p, qh, kvh = (c[n] for n in ("b", "t", "p", "qh", "kvh"))
    kv = _values(s["codes"], s["scales"])
    q = s["q"].float().view(b, t, kvh, qh // kvh, HD).permute(0, 2, 3, 1, 4).reshape(b, kvh, -1, HD)
    score = (q @ kv[:, 0].transpose(-1, -2).contiguous()).view(b, kvh, qh // kvh, t, p) / math.sqrt(HD)
    last = s["pos"].view(b, 1, 1, 1, 1) + torch.arange(t, device="cuda").view(t, 1)
    score = torch.where(torch.arange(p, device="cuda") <= last, score, -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    e = e / e.sum(-1, keepdim=True)
    o = (e.view(b, kvh, -1, p) @ kv[:, 1]).view(b, kvh, qh // kvh, t, HD)
    return o.permute(0, 3, 1, 2, 4).reshape(b * t, qh * HD).half()


def _plain_beam(s: dict, c: dict):
    x = s["logits"].double()  # candidates of different beams can be near each other
    top = x.amax(-1, keepdim=True)
    cand = s["scores"].double().unsqueeze(1) + (x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    token = torch.arange(c["v"], device="cuda")
    ended = torch.where(token == s["eos"], s["scores"].double().unsqueeze(1), -math.inf)
    cand = torch.where(s["done"].unsqueeze(1) > 0, ended, cand).flatten()
    score, at = torch.sort(torch.where(torch.isnan(cand), -math.inf, cand), descending=True, stable=True)
    score, at = score[: c["k"]], at[: c["k"]]
    parent, token = at // c["v"], at % c["v"]
    done = ((s["done"][parent] > 0) | (token == s["eos"])).long()
    s["codes"][..., : c["n"], :] = s["codes"][:, parent, ..., : c["n"], :]
    s["scales"][..., : c["n"], :] = s["scales"][:, parent, ..., : c["n"], :]
    return score.float(), parent, token, done, _values(s["codes"], s["scales"]).half()


def run(s: dict):
    c = s["case"]
    if own:
        lk, q4 = s["lk"], s["lk"].ops.q4_gpu
        if c["kind"] == "w4":
            x, w, epi = s["x"], s["w"], c["epi"]
            if epi == "swiglu":
                return q4.gemm_w4_swiglu_f16_gpu(x, w[0], w[1]).t
            if epi == "bias":
                return q4.gemm_w4_bias_f16_gpu(x, w[0], s["extra"]).t
            if epi == "add":
                return q4.gemm_w4_add_f16_gpu(x, w[0], s["extra"]).t
            return (q4.lm_head_w4_f16_gpu if epi == "logits" else q4.gemm_w4_f16_gpu)(x, w[0]).t
        if c["kind"] == "attn":
            return q4.attention_kv4_f16_gpu(s["q"], s["kv"], s["pos"]).t
        if c["kind"] == "fill":
            q4.kv4_write_f16_gpu(s["kv"], s["k"], s["v"], s["pos"])
            return q4.kv4_read_f16_gpu(s["kv"]).t[..., : c["t"], :]
        score, parent, token, done = lk.ops.beam_select_f32_gpu(s["logits"], s["scores"], s["done"], c["k"], eos=(s["eos"],))
        q4.kv4_reorder_gpu(s["kv"], parent, s["n"])
        return score.t, parent.t, token.t, done.t, q4.kv4_read_f16_gpu(s["kv"]).t[..., : c["p"], :]
    if c["kind"] == "w4":
        return _plain_w4(s, c)
    if c["kind"] == "attn":
        return _plain_attn(s, c)
    if c["kind"] == "fill":
        return _values(*_rows_q4(s["k"], s["v"], c["kvh"])).half()
    return _plain_beam(s, c)


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case: dict) -> dict:
    c = case
    if c["kind"] == "w4":
        m, k, n, two = c["m"], c["k"], c["n"], 2 if c["epi"] == "swiglu" else 1
        extra = {"bias": 2 * n, "add": 2 * m * n}.get(c["epi"], 0)
        weights = two * (n * k // 2 + 2 * n * -(-k // c["group"]))
        return {"bytes": weights + 2 * m * k + extra + m * n * (4 if c["epi"] == "logits" else 2), "flops": 2 * m * k * n * two}
    if c["kind"] == "attn":
        # the first sequence sees the whole cache, the others half of it in the mean
        b, t, p = c["b"], c["t"], c["p"]
        rows = p + (b - 1) * (p + t) // 2
        pairs = t * (p - t) + t * (t + 1) // 2
        pairs += (b - 1) * (t * (p - t) // 2 + t * (t + 1) // 2)
        return {"bytes": rows * c["kvh"] * 144 + 4 * b * t * c["qh"] * HD, "flops": 4 * pairs * HD * c["qh"]}
    if c["kind"] == "fill":
        rows = c["b"] * c["t"] * c["kvh"] * 2
        return {"bytes": rows * (256 + 2 * 72 + 256), "flops": 4 * rows * HD}
    # logits read once; the caches of beams with another parent (about half of them) read and written, then read as values
    rows = c["layers"] * c["b"] * 2 * c["kvh"]
    return {"bytes": 4 * c["b"] * c["v"] + rows * c["n"] * 72 + rows * c["p"] * (72 + 256), "flops": 4 * c["b"] * c["v"]}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_rows(k: torch.Tensor, v: torch.Tensor, kvh: int) -> torch.Tensor:
    """Values f64[B, 2, kvh, P, 128] that the quantised rows stand for: each group of 32 over its own scale."""
    x = torch.stack([k, v], 1).double()
    x = x.view(*x.shape[:3], kvh, 4, 32)
    need = torch.maximum(x.amax(-1) / 7, x.amin(-1) / -8).clamp(min=0).float().double()  # a quotient in 24 bits
    lift = torch.exp2(7 - torch.floor(torch.log2(need.clamp(min=2.0 ** -17))))  # 8 significant bits, or 2^-24
    s = (torch.ceil(need * lift) / lift).clamp(max=8128).unsqueeze(-1)
    c = torch.where(s > 0, torch.floor(x / s.clamp(min=2.0 ** -24) + 0.5), 0.0).clamp(-8, 7)
    return (c * s).flatten(-2).transpose(2, 3)


def exact(case: dict, seed: int):
    s, c = _inputs(case, seed), case
    if c["kind"] == "w4":
        ys = []
        for codes, scales in s["w"]:
            y = torch.zeros(c["m"], c["n"], dtype=torch.float64, device="cuda")
            for j in range(scales.shape[0]):  # group by group
                at = slice(j * c["group"], min((j + 1) * c["group"], c["k"]))
                y += (s["x"][:, at].double() @ (codes[at].double() - 8)) * scales[j].double()
            ys.append(y)
        if c["epi"] == "swiglu":
            return ys[0] * torch.sigmoid(ys[0]) * ys[1]
        return ys[0] + s["extra"].double() if c["epi"] in ("bias", "add") else ys[0]
    if c["kind"] == "fill":
        return _exact_rows(s["k"], s["v"], c["kvh"])
    if c["kind"] == "attn":
        kv, t, group = _exact_rows(s["k"], s["v"], c["kvh"]), c["t"], c["qh"] // c["kvh"]
        q = s["q"].double().view(c["b"], t, c["qh"], HD)
        out = torch.zeros_like(q)
        for b, p0 in enumerate(s["pos"].tolist()):
            seen = torch.arange(p0 + t, device="cuda") <= p0 + torch.arange(t, device="cuda").unsqueeze(1)
            for h in range(c["qh"]):
                key, value = kv[b, :, h // group, : p0 + t]
                logit = (q[b, :, h] @ key.T / math.sqrt(HD)).masked_fill(~seen, -math.inf)
                out[b, :, h] = torch.softmax(logit, -1) @ value
        return out.view(c["b"] * t, -1)
    lp = s["scores"].double().unsqueeze(1) + torch.log_softmax(s["logits"].double(), -1)
    for b in torch.nonzero(s["done"]).flatten().tolist():
        lp[b] = -math.inf
        lp[b, s["eos"]] = s["scores"][b]
    at = torch.argsort(lp.flatten(), descending=True, stable=True)[: c["k"]]
    parent, token = torch.div(at, c["v"], rounding_mode="floor"), at.remainder(c["v"])
    kv = torch.stack([_exact_rows(k, v, c["kvh"]) for k, v in s["rows"]])
    moved = kv.clone()
    moved[..., : c["n"], :] = kv.index_select(1, parent)[..., : c["n"], :]
    return lp.flatten()[at], parent, token, s["done"][parent] | (token == s["eos"]), moved
