"""Four operators of a batch that decodes over one shared, bounded cache: what is measured of them.

  rope    q / k norm and a rotation by several position axes, the new rows written at slots of their own
  shared  attention of many rows over one common prefix and each row's own keys, with the rows' log-sum-exp
  mass    the attention weight every cached key received from a pass, added to what it had
  evict   the cache cut to its heaviest keys, with the first and the newest kept

`listed` holds the cases, `draw` makes more of the same ranges; `run` is one pass in plain torch or, where `own` is set, through
`HipCard`; `exact` is the definition in 64 bits.
"""

from __future__ import annotations

import math
import random
from typing import Any

import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 1_000_000.0


def listed() -> list[dict[str, Any]]:
    return [
        # the next token of one conversation over a cache whose slots are no longer its positions: latency alone
        {"name": "rope_step", "kind": "rope", "T": 1, "Hq": 32, "Hk": 8, "D": 128, "A": 1, "table": "bf16", "mix": "runs",
         "norm": 1, "centered": 0, "layout": "head"},
        # a small vision model's forks: narrow heads, three axes dealt round in turn, full-precision tables
        {"name": "rope_forks", "kind": "rope", "T": 93, "Hq": 14, "Hk": 2, "D": 64, "A": 3, "table": "f32", "mix": "turns",
         "norm": 1, "centered": 0, "layout": "slot"},
        # a prompt of text and pictures: time, height and width in runs of frequencies
        {"name": "rope_prompt", "kind": "rope", "T": 16384, "Hq": 32, "Hk": 8, "D": 128, "A": 3, "table": "bf16", "mix": "runs",
         "norm": 1, "centered": 0, "layout": "head"},
        # four samples of a short prompt, a few tokens in: latency
        {"name": "shared_few", "kind": "shared", "T": 4, "Hq": 32, "Hk": 8, "D": 128, "P": 700, "own": 5, "layout": "head"},
        # forty users behind one system prompt, each with a question of their own; five query heads a kv head, narrow
        {"name": "shared_ragged", "kind": "shared", "T": 41, "Hq": 40, "Hk": 8, "D": 64, "P": 6001, "own": 777,
         "layout": "slot"},
        # sixteen samples over a long document: the keys' trip from memory
        {"name": "shared_long", "kind": "shared", "T": 16, "Hq": 32, "Hk": 8, "D": 128, "P": 131072, "own": 100,
         "layout": "head"},
        # a full serving batch behind a long prefix: the matrix cores' work
        {"name": "shared_wide", "kind": "shared", "T": 256, "Hq": 32, "Hk": 8, "D": 128, "P": 32768, "own": 1024,
         "layout": "head"},
        # the weight of one step over a full cache: the keys' trip from memory again
        {"name": "mass_step", "kind": "mass", "T": 4, "Hq": 32, "Hk": 8, "D": 128, "n": 32000, "chain": 1, "layout": "head"},
        # a chunk of a prompt, each of its rows over the keys before it: the matrix cores and the exponentials
        {"name": "mass_chunk", "kind": "mass", "T": 500, "Hq": 32, "Hk": 8, "D": 128, "n": 16384, "chain": 1,
         "layout": "head"},
        # one layer's short cache cut once: latency
        {"name": "evict_short", "kind": "evict", "L": 1, "Hk": 8, "D": 128, "n": 700, "budget": 512, "sinks": 4, "recent": 64,
         "ties": 0, "mixed": 0},
        # every layer of the stack back to its budget, again after earlier cuts
        {"name": "evict_stack", "kind": "evict", "L": 36, "Hk": 8, "D": 128, "n": 4608, "budget": 4096, "sinks": 4,
         "recent": 256, "ties": 1, "mixed": 1},
        # a long document's keys down to an eighth, right after the prompt
        {"name": "evict_document", "kind": "evict", "L": 4, "Hk": 8, "D": 128, "n": 131072, "budget": 16384, "sinks": 4,
         "recent": 1024, "ties": 1, "mixed": 0},
    ]


def _log(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng: random.Random) -> dict[str, Any]:
    kind = rng.choice(["rope", "shared", "shared", "mass", "evict"])
    Hk = rng.choice([1, 2, 3, 4, 8])
    layout = rng.choice(["head", "slot"])
    if kind == "rope":
        Hq, D = Hk * rng.randint(1, 8), rng.choice([64, 128, 256])
        T = _log(rng, 1, max(1, min(16384, 16384 * 48 * 128 // ((Hq + 2 * Hk) * D))))
        return {"kind": kind, "T": T, "Hq": Hq, "Hk": Hk, "D": D, "A": rng.randint(1, 4), "table": rng.choice(["bf16", "f32"]),
                "mix": rng.choice(["runs", "turns"]), "norm": int(rng.random() < 0.8), "centered": int(rng.random() < 0.2),
                "layout": layout}
    if kind == "shared":
        Hq, D, T, own_keys = Hk * rng.randint(1, 8), rng.choice([64, 128]), _log(rng, 1, 256), _log(rng, 1, 1024)
        P = _log(rng, 1, max(1, min(131072, 256 * 32 * 128 * 32768 // (T * Hq * D))))
        return {"kind": kind, "T": T, "Hq": Hq, "Hk": Hk, "D": D, "P": P, "own": own_keys, "layout": layout}
    if kind == "mass":
        Hq, D, T = Hk * rng.randint(1, 8), rng.choice([64, 128]), _log(rng, 1, 500)
        n = _log(rng, 1, max(1, min(131072, 500 * 32 * 128 * 16384 // (T * Hq * D))))
        return {"kind": kind, "T": T, "Hq": Hq, "Hk": Hk, "D": D, "n": n, "chain": rng.randint(0, 1), "layout": layout}
    L, D = _log(rng, 1, 36), rng.choice([64, 128])
    n = _log(rng, 2, max(2, min(131072, 4 * 8 * 131072 // (L * Hk))))
    return {"kind": kind, "L": L, "Hk": Hk, "D": D, "n": n, "budget": _log(rng, 1, n), "sinks": rng.randint(0, 8),
            "recent": rng.randint(0, max(1, n // 8)), "ties": rng.randint(0, 1), "mixed": rng.randint(0, 1)}


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _normal(g: torch.Generator, *shape: int, std: float = 1.0) -> torch.Tensor:
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def _cache(g: torch.Generator, layout: str, Hk: int, cap: int, D: int) -> torch.Tensor:
    """keys or values [Hk, cap, D]: a head's rows together, or (a view) a slot's heads together"""
    return _normal(g, Hk, cap, D) if layout == "head" else _normal(g, cap, Hk, D).transpose(0, 1)


def _axes(case: dict[str, Any]) -> list[int]:
    """which axis turns each of the D / 2 frequencies: in runs (the first a little shorter, as such models have it), or in turn"""
    half, A = case["D"] // 2, case["A"]
    if case["mix"] == "turns":
        return [i % A for i in range(half)]
    runs = [half // (2 * A) if a == 0 and A > 1 else 0 for a in range(A)]
    for a in range(A):
        if runs[a] == 0:
            runs[a] = (half - runs[0]) // (A - 1) if A > 1 else half
    runs[-1] += half - sum(runs)
    return [a for a in range(A) for _ in range(runs[a])]


def _rope_inputs(case: dict[str, Any], g: torch.Generator) -> dict[str, Any]:
    T, Hq, Hk, D, A = (case[k] for k in ("T", "Hq", "Hk", "D", "A"))
    table = 32768
    inv = 1.0 / (THETA ** (torch.arange(0, D // 2, dtype=torch.float32, device="cuda") * 2.0 / D))
    ang = torch.arange(table, dtype=torch.float32, device="cuda")[:, None] * inv[None, :]
    cos, sin = ang.cos(), ang.sin()
    if case["table"] == "bf16":  # the framework's tables: both halves of the dims, bf16
        cos, sin = (torch.cat([t, t], dim=-1).to(torch.bfloat16) for t in (cos, sin))
    # text stands at one place on every axis; about half of the rows are patches of pictures, 32 to a line
    start = int(torch.randint(0, 8192, (1,), generator=g, device="cuda"))
    t = torch.arange(T, device="cuda", dtype=torch.int32) + start
    picture = (t // 256) % 2 == 1
    place = [torch.where(picture, t // 256 * 256, t), torch.where(picture, t // 256 * 256 + (t % 256) // 32, t),
             torch.where(picture, t // 256 * 256 + t % 32, t), t // 2]
    cap = T + 77
    slots = torch.randperm(cap, generator=g, device="cuda")[:T].to(torch.int32)
    return {"qkv": _normal(g, T, (Hq + 2 * Hk) * D), "wq": (1.0 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16)
            if case["norm"] else None, "wk": (1.0 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16)
            if case["norm"] else None, "cos": cos.contiguous(), "sin": sin.contiguous(),
            "pos": torch.stack(place[:A]).to(torch.int32).contiguous(),
            "axes": torch.tensor(_axes(case), dtype=torch.uint8, device="cuda"), "slots": slots,
            "K": _cache(g, case["layout"], Hk, cap, D), "V": _cache(g, case["layout"], Hk, cap, D)}


def _own_lengths(case: dict[str, Any], seed: int) -> list[int]:
    """how many keys of its own each row has: between a quarter of `own` and all of it, as rows of unlike age have"""
    rng = random.Random(1_000_003 * int(seed) + case["T"])
    return [rng.randint(max(1, case["own"] // 4), case["own"]) for _ in range(case["T"])]


def _shared_inputs(case: dict[str, Any], g: torch.Generator, seed: int) -> dict[str, Any]:
    T, Hq, Hk, D, P = (case[k] for k in ("T", "Hq", "Hk", "D", "P"))
    lens = _own_lengths(case, seed)
    # the rows' own stretches around the prefix: half of them ahead of it, each with room to grow
    offs, at, off = [], 3, 0
    for t in range(T):
        if t == T // 2:
            off, at = at, at + P + 5
        offs.append(at)
        at += lens[t] + 2
    return {"q": _normal(g, T, Hq * D, std=1.5), "K": _cache(g, case["layout"], Hk, at, D),
            "V": _cache(g, case["layout"], Hk, at, D), "off": off, "offs": offs, "lens": lens, "scale": 1.0 / math.sqrt(D)}


def _mass_inputs(case: dict[str, Any], g: torch.Generator) -> dict[str, Any]:
    T, Hq, Hk, D, n = (case[k] for k in ("T", "Hq", "Hk", "D", "n"))
    q, K = _normal(g, T, Hq * D, std=1.5), _cache(g, case["layout"], Hk, n + 9, D)
    seen = torch.full((T,), n, dtype=torch.int32, device="cuda")
    if case["chain"]:
        seen = (seen - T + 1 + torch.arange(T, device="cuda", dtype=torch.int32)).clamp(min=1)
    scale = 1.0 / math.sqrt(D)
    # the rows' log-sum-exp, as the pass's attention leaves it
    hidden = torch.arange(n, device="cuda")[None, None, :] >= seen[:, None, None]
    scores = _scores(q, K[:, :n], case, scale).masked_fill_(hidden, -math.inf)
    lse = torch.logsumexp(scores, dim=-1).transpose(0, 1).reshape(T, Hq)
    mass = torch.rand(Hk, n + 9, generator=g, device="cuda") ** 4 * 8.0
    return {"q": q, "K": K, "lse": lse, "seen": seen, "mass": mass, "scale": scale}


def _evict_inputs(case: dict[str, Any], g: torch.Generator) -> dict[str, Any]:
    L, Hk, D, n = (case[k] for k in ("L", "Hk", "D", "n"))
    # few keys hold most of the weight; under `ties` many hold none and others the same
    mass = torch.exp(2.0 * torch.randn(L, Hk, n, generator=g, device="cuda"))
    if case["ties"]:
        mass = torch.where(mass < 1.0, torch.zeros_like(mass), torch.round(mass * 16.0) / 16.0)
    pos = torch.arange(n, dtype=torch.int32, device="cuda").expand(L, Hk, n)
    if case["mixed"]:  # earlier cuts have moved the older keys about, each head's in its own way
        old = n * 7 // 8
        mixed = torch.rand(L, Hk, old, generator=g, device="cuda").argsort(dim=-1).to(torch.int32)
        pos = torch.cat([mixed, pos[..., old:]], dim=-1)
    return {"mass": mass.contiguous(), "pos": pos.contiguous(), "K": _normal(g, L, Hk, n, D), "V": _normal(g, L, Hk, n, D)}


def _inputs(case: dict[str, Any], seed: int) -> dict[str, Any]:
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["kind"] == "shared":
        return _shared_inputs(case, g, seed)
    return {"rope": _rope_inputs, "mass": _mass_inputs, "evict": _evict_inputs}[case["kind"]](case, g)


def prepare(case: dict[str, Any], seed: int) -> dict[str, Any]:
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if kind == "shared" and not own:
        s["lay"] = (torch.tensor(s["offs"], device="cuda"), torch.tensor(s["lens"], device="cuda"))
    if not own:
        return s
    from btb_amd.native import Native

    card = s["card"] = Native.card_kernels()
    if kind == "rope":
        s["q"] = torch.zeros(case["T"], case["Hq"] * case["D"], dtype=torch.bfloat16, device="cuda")
    elif kind == "shared":
        T, Hq, Hk, D, P = (case[k] for k in ("T", "Hq", "Hk", "D", "P"))
        s["lay"] = card.shared_layout(s["off"], P, list(zip(s["offs"], s["lens"])))
        s["att"] = torch.zeros(T, Hq * D, dtype=torch.bfloat16, device="cuda")
        s["lse"] = torch.zeros(T, Hq, dtype=torch.float32, device="cuda")
        s["scratch"] = card.attn_shared_scratch(T, Hq, Hk, D, P, case["own"])
    elif kind == "mass":
        s["out"] = torch.zeros_like(s["mass"])
    else:
        L, Hk, D, kept = case["L"], case["Hk"], case["D"], min(case["n"], case["budget"])
        for k in ("K", "V"):
            s[k + "_out"] = torch.zeros(L, Hk, kept, D, dtype=torch.bfloat16, device="cuda")
        s["mass_out"] = torch.zeros(L, Hk, kept, dtype=torch.float32, device="cuda")
        s["pos_out"] = torch.zeros(L, Hk, kept, dtype=torch.int32, device="cuda")
        s["idx"] = torch.zeros(L, Hk, kept, dtype=torch.int32, device="cuda")
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------


def run(s: dict[str, Any]) -> Any:
    kind = s["case"]["kind"]
    if own:
        return {"rope": _own_rope, "shared": _own_shared, "mass": _own_mass, "evict": _own_evict}[kind](s)
    return {"rope": _plain_rope, "shared": _plain_shared, "mass": _plain_mass, "evict": _plain_evict}[kind](s)


def _own_rope(s: dict[str, Any]) -> Any:
    c = s["case"]
    s["card"].norm_rope_axes(s["qkv"], s["wq"], s["wk"], EPS, s["cos"], s["sin"], s["pos"], s["axes"], s["slots"], s["K"], s["V"],
                             s["q"], c["Hq"], c["Hk"], c["D"], centered=bool(c["centered"]))
    return s["q"], s["K"], s["V"]


def _own_shared(s: dict[str, Any]) -> Any:
    c = s["case"]
    s["card"].attn_shared(s["q"], s["K"], s["V"], s["att"], s["lay"], c["Hq"], c["Hk"], c["D"], s["scale"], c["P"], c["own"],
                          s["scratch"], lse=s["lse"])
    return s["att"], s["lse"]


def _own_mass(s: dict[str, Any]) -> Any:
    c = s["case"]
    s["card"].attn_mass(s["q"], s["K"], s["lse"], s["seen"], s["mass"], c["Hq"], c["Hk"], c["D"], s["scale"], c["n"], out=s["out"])
    return s["out"][:, :c["n"]]


def _own_evict(s: dict[str, Any]) -> Any:
    c = s["case"]
    s["card"].kv_evict(s["mass"], s["pos"], s["K"], s["V"], c["n"], c["budget"], s["K_out"], s["V_out"], s["mass_out"], s["pos_out"],
                       s["idx"], sinks=c["sinks"], recent_from=c["n"] - c["recent"])
    return s["idx"], s["K_out"], s["V_out"], s["mass_out"], s["pos_out"]


def _plain_rope(s: dict[str, Any]) -> Any:
    c = s["case"]
    T, Hq, Hk, D = (c[k] for k in ("T", "Hq", "Hk", "D"))
    half = D // 2
    heads = s["qkv"].view(T, Hq + 2 * Hk, D)
    which = s["pos"].long().t()[:, s["axes"].long()]  # [T, D / 2]: the place each frequency turns by
    cos, sin = (s[k][:, :half].float().gather(0, which)[:, None, :] for k in ("cos", "sin"))

    def turned(x: torch.Tensor, w: torch.Tensor | None) -> torch.Tensor:
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * (w.float() + 1.0 if c["centered"] else w.float())
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(torch.bfloat16)

    at = s["slots"].long()
    s["K"][:, at] = turned(heads[:, Hq:Hq + Hk], s["wk"]).transpose(0, 1)
    s["V"][:, at] = heads[:, Hq + Hk:].transpose(0, 1)
    return turned(heads[:, :Hq], s["wq"]).reshape(T, Hq * D), s["K"], s["V"]


def _scores(q: torch.Tensor, K: torch.Tensor, c: dict[str, Any], scale: float) -> torch.Tensor:
    """the scores [Hk, T, G, keys] in 32 bits"""
    T, Hk, D = c["T"], c["Hk"], c["D"]
    rows = q.view(T, Hk, -1, D).transpose(0, 1).float().reshape(Hk, -1, D) * scale
    return torch.matmul(rows, K.float().transpose(1, 2)).view(Hk, T, -1, K.shape[1])


def _plain_shared(s: dict[str, Any]) -> Any:
    c = s["case"]
    T, Hq, Hk, D, P = (c[k] for k in ("T", "Hq", "Hk", "D", "P"))
    off = s["off"]
    first, lens = s["lay"]
    step = torch.arange(c["own"], device="cuda")
    at = first[:, None] + torch.minimum(step[None, :], lens[:, None] - 1)  # [T, own], a row's last key again past its end
    past = (step[None, :] >= lens[:, None])[:, None, :]
    far = _scores(s["q"], s["K"][:, off:off + P], c, s["scale"])
    rows = s["q"].view(T, Hk, -1, D).transpose(0, 1).float() * s["scale"]
    near = torch.matmul(rows, s["K"][:, at].float().transpose(2, 3)).masked_fill_(past, -math.inf)
    top = torch.maximum(far.amax(dim=-1), near.amax(dim=-1))
    far, near = far.sub_(top[..., None]).exp_(), near.sub_(top[..., None]).exp_()
    total = far.sum(dim=-1) + near.sum(dim=-1)
    out = torch.matmul(far.view(Hk, -1, P), s["V"][:, off:off + P].float()).view(rows.shape)
    out = (out + torch.matmul(near, s["V"][:, at].float())) / total[..., None]
    return (out.to(torch.bfloat16).transpose(0, 1).reshape(T, Hq * D), (top + torch.log(total)).transpose(0, 1).reshape(T, Hq))


def _plain_mass(s: dict[str, Any]) -> Any:
    c = s["case"]
    n = c["n"]
    hidden = torch.arange(n, device="cuda")[None, None, :] >= s["seen"][:, None, None]
    lse = s["lse"].view(c["T"], c["Hk"], -1).transpose(0, 1)[..., None]
    p = _scores(s["q"], s["K"][:, :n], c, s["scale"]).sub_(lse).exp_()
    return s["mass"][:, :n] + p.masked_fill_(hidden, 0.0).sum(dim=(1, 2))


def _plain_evict(s: dict[str, Any]) -> Any:
    c = s["case"]
    n, kept = c["n"], min(c["n"], c["budget"])
    held = (s["pos"] < c["sinks"]) | (s["pos"] >= n - c["recent"])
    rank = torch.where(held, math.inf, torch.where(torch.isnan(s["mass"]), -math.inf, s["mass"] + 0.0))
    first = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :kept]
    stays = torch.zeros(rank.shape, dtype=torch.bool, device="cuda").scatter_(-1, first, True)
    idx = torch.arange(kept, device="cuda").expand(c["L"], c["Hk"], kept).clone()
    # a head has as many kept keys past the end as holes before it: both in ascending order, a head after the other
    idx[~stays[..., :kept]] = stays[..., kept:].nonzero()[:, 2] + kept
    rows = idx[..., None].expand(-1, -1, -1, c["D"])
    return (idx.to(torch.int32), s["K"].gather(2, rows), s["V"].gather(2, rows), s["mass"].gather(2, idx),
            s["pos"].gather(2, idx))


def work(case: dict[str, Any]) -> dict[str, float]:
    c, kind = case, case["kind"]
    if kind == "rope":
        values = c["T"] * (c["Hq"] + 2 * c["Hk"]) * c["D"]
        tables = c["T"] * c["D"] * (2 if c["table"] == "bf16" else 4)  # D / 2 cosines and as many sines a row
        return {"bytes": 4.0 * values + tables + 4.0 * c["T"] * (c["A"] + 1), "flops": 8.0 * values}
    if kind == "shared":
        mean = (max(1, c["own"] // 4) + c["own"]) / 2.0
        keys = c["P"] + c["T"] * mean
        return {"bytes": 4.0 * c["Hk"] * c["D"] * keys + 4.0 * c["T"] * c["Hq"] * (c["D"] + 1),
                "flops": 4.0 * c["T"] * c["Hq"] * c["D"] * (c["P"] + mean)}
    if kind == "mass":
        return {"bytes": 2.0 * c["Hk"] * c["D"] * c["n"] + 2.0 * c["T"] * c["Hq"] * (c["D"] + 2) + 8.0 * c["Hk"] * c["n"],
                "flops": 2.0 * c["T"] * c["Hq"] * c["D"] * (c["n"] - (c["T"] // 2 if c["chain"] and c["T"] < c["n"] else 0))}
    kept = min(c["n"], c["budget"])
    return {"bytes": c["L"] * c["Hk"] * (8.0 * c["n"] + kept * (8.0 * c["D"] + 20.0)), "flops": 0.0}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------


def exact(case: dict[str, Any], seed: int) -> Any:
    s = _inputs(case, seed)
    return {"rope": _exact_rope, "shared": _exact_shared, "mass": _exact_mass, "evict": _exact_evict}[case["kind"]](case, s)


def _exact_rope(c: dict[str, Any], s: dict[str, Any]) -> Any:
    T, Hq, Hk, D = (c[k] for k in ("T", "Hq", "Hk", "D"))
    half = D // 2
    x = s["qkv"].double().view(T, Hq + 2 * Hk, D)
    cos, sin = (torch.empty(T, 1, half, dtype=torch.float64, device="cuda") for _ in range(2))
    for i, a in enumerate(_axes(c)):
        cos[:, 0, i] = s["cos"][s["pos"][a].long(), i].double()
        sin[:, 0, i] = s["sin"][s["pos"][a].long(), i].double()
    K, V = s["K"].double(), s["V"].double()
    out = torch.empty(T, Hq + Hk, D, dtype=torch.float64, device="cuda")
    for heads, w in ((slice(0, Hq), s["wq"]), (slice(Hq, Hq + Hk), s["wk"])):
        y = x[:, heads]
        if w is not None:
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / D + EPS) * (w.double() + c["centered"])
        out[:, heads, :half] = y[..., :half] * cos - y[..., half:] * sin
        out[:, heads, half:] = y[..., half:] * cos + y[..., :half] * sin
    for t, slot in enumerate(s["slots"].tolist()):
        K[:, slot], V[:, slot] = out[t, Hq:], x[t, Hq + Hk:]
    return out[:, :Hq].reshape(T, Hq * D), K, V


def _exact_shared(c: dict[str, Any], s: dict[str, Any]) -> Any:
    T, Hq, Hk, D, P = (c[k] for k in ("T", "Hq", "Hk", "D", "P"))
    G, off = Hq // Hk, s["off"]
    out = torch.empty(T, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.empty(T, Hq, dtype=torch.float64, device="cuda")
    q = s["q"].double().view(T, Hq, D)
    for h in range(Hk):
        K, V = s["K"][h].double(), s["V"][h].double()
        heads = slice(h * G, (h + 1) * G)
        rows = q[:, heads].reshape(T * G, D)
        z_far, o_far = [], []
        for i in range(0, T * G, 256):  # a few rows at a time: their scores in 64 bits are 2 KB a key
            a = rows[i:i + 256] @ K[off:off + P].T * s["scale"]
            z = torch.logsumexp(a, -1)
            z_far.append(z)
            o_far.append(torch.exp(a - z[:, None]) @ V[off:off + P])
        z_far, o_far = torch.cat(z_far).view(T, G), torch.cat(o_far).view(T, G, D)
        for t in range(T):
            mine = slice(s["offs"][t], s["offs"][t] + s["lens"][t])
            b = q[t, heads] @ K[mine].T * s["scale"]
            zb = torch.logsumexp(b, -1)
            z = torch.logaddexp(z_far[t], zb)
            out[t, heads] = o_far[t] * torch.exp(z_far[t] - z)[:, None] + torch.exp(b - z[:, None]) @ V[mine]
            lse[t, heads] = z
    return out.view(T, Hq * D), lse


def _exact_mass(c: dict[str, Any], s: dict[str, Any]) -> Any:
    T, Hq, Hk, D, n = (c[k] for k in ("T", "Hq", "Hk", "D", "n"))
    G = Hq // Hk
    out = s["mass"][:, :n].double()
    q, lse, seen = s["q"].double().view(T, Hq, D), s["lse"].double(), s["seen"].tolist()
    for h in range(Hk):
        K = s["K"][h, :n].double()
        for t in range(0, T, 32):
            a = q[t:t + 32, h * G:(h + 1) * G] @ K.T * s["scale"]
            w = torch.exp(a - lse[t:t + 32, h * G:(h + 1) * G, None])
            for i in range(w.shape[0]):
                w[i, :, seen[t + i]:] = 0.0
            out[h] += w.sum((0, 1))
    return out


def _exact_evict(c: dict[str, Any], s: dict[str, Any]) -> Any:
    n, kept = c["n"], min(c["n"], c["budget"])
    mass, pos = s["mass"].cpu().numpy().reshape(-1, n), s["pos"].cpu().numpy().reshape(-1, n)
    idx = np.empty((mass.shape[0], kept), np.int64)
    for r in range(mass.shape[0]):
        m = mass[r].astype(np.float64)
        m[np.isnan(m)] = -np.inf
        m[(pos[r] < c["sinks"]) | (pos[r] >= n - c["recent"])] = np.inf
        chosen = np.zeros(n, bool)
        chosen[np.lexsort((np.arange(n), -m))[:kept]] = True
        late = iter(np.flatnonzero(chosen[kept:]) + kept)
        idx[r] = [j if chosen[j] else next(late) for j in range(kept)]
    at = torch.from_numpy(idx).cuda().view(c["L"], c["Hk"], kept)
    layer, head = torch.arange(c["L"], device="cuda")[:, None, None], torch.arange(c["Hk"], device="cuda")[None, :, None]
    return (at.to(torch.int32), s["K"][layer, head, at].double(), s["V"][layer, head, at].double(), s["mass"][layer, head, at].double(),
            s["pos"][layer, head, at])
