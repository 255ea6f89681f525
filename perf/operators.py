"""Timed cases of the KV-cache operators (``s2hip.KvOps``): what a program that
serves many requests over device-resident caches calls per layer.

* ``append`` -- head norms and position rotation of the new tokens' queries and
  keys in one pass, keys and values written to the requests' cache slots.
* ``attend`` -- attention of a batch whose requests share one long prefix (a
  voice-clone prompt): each request's new tokens see the prefix and the
  request's own cached tokens.
* ``weigh``  -- the same with every key's attention weight, summed over the
  query heads of its group and the new tokens, added to its score.
* ``evict``  -- a cache cut down to ``keep`` tokens by those scores; the first
  ``sinks`` and the last ``recent`` positions stay, kept rows behind the cut
  move into the freed slots before it.

With ``own`` false, ``run`` computes them from elementary torch operations in
float32 (angles in float64); with ``own`` true it calls the framework.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

ROPE_BASE = 1.0e6
EPS = 1.0e-6
TYPES = {"f32": torch.float32, "f16": torch.float16}


def listed():
    return [
        # three requests after a short shared text on the small model's heads: launch latency
        {"name": "prefix_step_3", "op": "attend", "requests": 3, "tokens": 1, "prefix": 100, "slots": 20, "cap": 64, "heads": 8, "kv_heads": 2, "hd": 64, "type": "f32"},
        # eight voice-clone requests, one decode step over the 1500-position prompt they share
        {"name": "prefix_step_8", "op": "attend", "requests": 8, "tokens": 1, "prefix": 1500, "slots": 512, "cap": 768, "heads": 32, "kv_heads": 8, "hd": 128, "type": "f32"},
        # sixteen requests late in long sessions over a very long prompt, half-precision caches
        {"name": "prefix_step_16_long", "op": "attend", "requests": 16, "tokens": 1, "prefix": 24001, "slots": 2000, "cap": 2048, "heads": 32, "kv_heads": 8, "hd": 128, "type": "f16"},
        # eight requests bring a turn of text each (ragged) over the shared voice prompt
        {"name": "prefix_turn_8", "op": "attend", "requests": 8, "tokens": 250, "prefix": 1500, "slots": 250, "cap": 768, "heads": 32, "kv_heads": 8, "hd": 128, "type": "f16"},
        # an odd turn of three requests on f32 caches that hold earlier turns
        {"name": "prefix_turn_3", "op": "attend", "requests": 3, "tokens": 37, "prefix": 1001, "slots": 131, "cap": 768, "heads": 32, "kv_heads": 8, "hd": 128, "type": "f32"},
        # decode steps of eight requests that keep scores over their own prompts
        {"name": "weigh_step_8", "op": "weigh", "requests": 8, "tokens": 1, "prefix": 0, "slots": 1509, "cap": 2560, "heads": 32, "kv_heads": 8, "hd": 128, "type": "f32"},
        # long sessions: four requests, shared prompt scored too, half-precision caches
        {"name": "weigh_step_4_long", "op": "weigh", "requests": 4, "tokens": 1, "prefix": 1500, "slots": 20000, "cap": 32768, "heads": 32, "kv_heads": 8, "hd": 128, "type": "f16"},
        # a whole voice-clone prompt scores itself before the first eviction
        {"name": "weigh_prompt", "op": "weigh", "requests": 1, "tokens": 1500, "prefix": 0, "slots": 1500, "cap": 2560, "heads": 32, "kv_heads": 8, "hd": 128, "type": "f16"},
        # one decode step of eight requests: launch latency
        {"name": "append_step_8", "op": "append", "requests": 8, "tokens": 1, "slots": 512, "cap": 768, "heads": 32, "kv_heads": 8, "hd": 128, "type": "f32"},
        # the turn of eight requests
        {"name": "append_turn_8", "op": "append", "requests": 8, "tokens": 250, "slots": 250, "cap": 768, "heads": 32, "kv_heads": 8, "hd": 128, "type": "f16"},
        # one layer of eight full caches cut to 1024 tokens
        {"name": "evict_8", "op": "evict", "requests": 8, "layers": 1, "slots": 2560, "cap": 2560, "keep": 1024, "recent": 256, "sinks": 4, "kv_heads": 8, "hd": 128, "type": "f32", "shuffled": False},
        # every layer of four requests at once, caches that were cut before
        {"name": "evict_4_layers", "op": "evict", "requests": 4, "layers": 36, "slots": 1999, "cap": 2048, "keep": 777, "recent": 128, "sinks": 4, "kv_heads": 8, "hd": 128, "type": "f16", "shuffled": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "weigh", "weigh", "append", "evict"])
    heads, kv_heads, hd = rng.choice([(32, 8, 128), (32, 8, 128), (8, 2, 64), (16, 16, 64), (24, 8, 128), (14, 2, 128)])
    c = {"op": op, "requests": _log_int(rng, 1, 16), "kv_heads": kv_heads, "hd": hd, "type": rng.choice(["f32", "f16"])}
    if op == "evict":
        slots = _log_int(rng, 40, 2500)
        keep = rng.randint(slots // 4 + 4, slots)
        return dict(c, layers=rng.choice([1, 1, 4]), slots=slots, cap=slots + rng.randint(0, 200), keep=keep,
                    recent=rng.randint(0, keep // 2), sinks=rng.randint(0, 4), shuffled=rng.random() < 0.5)
    c["heads"] = heads
    if rng.random() < 0.5:
        c["tokens"] = rng.choice([1, 1, 2, 3, 4])
        c["slots"] = c["tokens"] - 1 + _log_int(rng, 1, 3000)
    else:
        c["requests"] = min(c["requests"], 8)
        c["tokens"] = _log_int(rng, 5, 1500 // c["requests"])
        c["slots"] = c["tokens"] + rng.choice([0, 0, _log_int(rng, 1, 500)])
    c["cap"] = c["slots"] + rng.randint(0, 300)
    if op != "append":
        c["prefix"] = rng.choice([0, _log_int(rng, 1, 6000)]) if op == "weigh" else _log_int(rng, 1, 6000)
        if c["tokens"] > 4:
            c["prefix"] = min(c["prefix"], 1500)
    return c


def _ragged(case):
    """(new tokens, slots in use) of each request; the new tokens are the last slots."""
    n, s, r = case.get("tokens", 0), case["slots"], case["requests"]
    new = [n - (b * 29) % (n // 2 + 1) for b in range(r)]
    used = [max(new[b], s - b * (s // (2 * r))) for b in range(r)]
    return new, used


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _inputs(case, seed):
    """The tensors of a case, from its seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 2 + 1)

    def normal(*shape, spread=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(spread)

    dt = TYPES[case["type"]]
    r, g_, hd, cap = case["requests"], case["kv_heads"], case["hd"], case["cap"]
    new, used = _ragged(case)
    s = {"lens": torch.tensor(used, dtype=torch.int32, device="cuda")}
    layers = case.get("layers", 1)
    # caches are allocated once and hold what earlier tokens left in slots not in use
    s["k"] = normal(layers * r, g_, cap, hd).to(dt)
    s["v"] = normal(layers * r, g_, cap, hd).to(dt)
    if case["op"] == "evict":
        # accumulated weights: few heavy tokens, many light ones, some never attended
        score = torch.exp(normal(layers * r, g_, cap, spread=2.0))
        s["scores"] = torch.where(normal(layers * r, g_, cap) > 1.3, torch.zeros_like(score), score)
        pos = torch.arange(cap, dtype=torch.int32, device="cuda").expand(layers * r, g_, cap)
        if case["shuffled"]:  # an earlier cut left the slots out of order
            order = torch.rand(layers * r, g_, cap, generator=g, device="cuda")
            out = torch.arange(cap, device="cuda") >= s["lens"].repeat(layers)[:, None, None]
            pos = torch.argsort(order + 2.0 * out, dim=2).to(torch.int32)
        s["positions"] = pos.contiguous()
        s["scores_out"] = torch.full_like(s["scores"], -1.0)
        s["positions_out"] = torch.full_like(s["positions"], -1)
        s["lens_out"] = torch.zeros_like(s["lens"])
        return s
    n, h = case["tokens"], case["heads"]
    s["new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
    if case["op"] == "append":
        s["qkv"] = normal(r, n, (h + 2 * g_) * hd, spread=3.0)
        s["q_norm"] = normal(hd, spread=0.2).add_(1.0)
        s["k_norm"] = normal(hd, spread=0.2).add_(1.0)
        first = torch.randint(0, 30000, (r, 1), generator=g, device="cuda")  # positions run ahead of the slots after cuts
        s["positions"] = (first + torch.arange(n, device="cuda")).to(torch.int32)
        s["q"] = torch.zeros(r, n, h * hd, device="cuda")
        s["scores"] = normal(r, g_, cap).abs_()
        s["slot_positions"] = torch.zeros(r, g_, cap, dtype=torch.int32, device="cuda")
        return s
    # normed and rotated queries, their gains a little over one: scores spread by about 1.5
    s["q"] = normal(r, n, h * hd, spread=1.5)
    s["out"] = torch.zeros(r, n, h * hd, device="cuda")
    p = case["prefix"]
    if p:
        s["prefix_k"] = normal(g_, p, hd).to(dt)
        s["prefix_v"] = normal(g_, p, hd).to(dt)
    if case["op"] == "weigh":
        s["weights"] = normal(r, g_, cap, spread=0.05).abs_()
        s["weights_out"] = torch.zeros(r, g_, cap, device="cuda")
        if p:
            s["prefix_weights"] = normal(g_, p, spread=0.05).abs_()
            s["prefix_weights_out"] = torch.zeros(g_, p, device="cuda")
    return s


_opened = {}


def _ops(case):
    """The handle of these heads: a program keeps it as long as its model."""
    key = (case.get("heads", case["kv_heads"]), case["kv_heads"], case["hd"], case["type"])
    if key not in _opened:
        sys.path.insert(0, os.path.abspath("fish-s2pro_amd"))
        from s2hip import KvOps

        _opened[key] = KvOps(key[0], key[1], key[2], max_requests=16, max_tokens=2048, kv_f16=key[3] == "f16", rope_base=ROPE_BASE, eps=EPS)
    return _opened[key]


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:  # the handle and the description of the caches, which a program keeps per layer
        ops = state["ops"] = _ops(case)
        at = lambda name: state[name].data_ptr() if name in state else 0  # noqa: E731
        state["view"] = ops.view(at("k"), at("v"), at("lens"), case["requests"], case["cap"], new_lens=at("new"), prefix_k=at("prefix_k"),
                                 prefix_v=at("prefix_v"), prefix_len=case.get("prefix", 0))
    return state


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def _run_own(s):
    c, ops, view = s["case"], s["ops"], s["view"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "append":
        ops.append(view, s["qkv"].data_ptr(), c["tokens"], s["positions"].data_ptr(), s["q"].data_ptr(), q_norm=s["q_norm"].data_ptr(),
                   k_norm=s["k_norm"].data_ptr(), scores=s["scores"].data_ptr(), slot_positions=s["slot_positions"].data_ptr(), stream=stream)
        return {k: s[k] for k in ("q", "k", "v", "scores", "slot_positions")}
    if c["op"] == "attend":
        ops.attend(view, s["q"].data_ptr(), c["tokens"], s["out"].data_ptr(), stream=stream)
        return s["out"]
    if c["op"] == "weigh":
        p = c["prefix"] > 0
        ops.attend_weigh(view, s["q"].data_ptr(), c["tokens"], s["out"].data_ptr(), s["weights_out"].data_ptr(), weights_in=s["weights"].data_ptr(),
                         prefix_weights_out=s["prefix_weights_out"].data_ptr() if p else 0,
                         prefix_weights_in=s["prefix_weights"].data_ptr() if p else 0, stream=stream)
        return {k: s[k] for k in ("out", "weights_out", "prefix_weights_out") if k in s}
    ops.evict(view, c["keep"], c["recent"], c["sinks"], s["scores"].data_ptr(), s["positions"].data_ptr(), s["scores_out"].data_ptr(),
              s["positions_out"].data_ptr(), s["lens_out"].data_ptr(), layers=c["layers"], stream=stream)
    return {k: s[k] for k in ("k", "v", "scores_out", "positions_out", "lens_out")}


def _plain_append(s):
    c = s["case"]
    r, n, h, g, hd, cap = c["requests"], c["tokens"], c["heads"], c["kv_heads"], c["hd"], c["cap"]
    x = s["qkv"].view(r, n, h + 2 * g, hd)

    def rotated(x, gain):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain
        freq = ROPE_BASE ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
        angle = s["positions"].double()[:, :, None, None] * freq
        cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).reshape(x.shape)

    live = torch.arange(n, device="cuda") < s["new"][:, None]
    slot = (s["lens"] - s["new"])[:, None] + torch.arange(n, device="cuda")
    req, tok = live.nonzero(as_tuple=True)
    at = slot[req, tok]
    q = rotated(x[:, :, :h], s["q_norm"]).reshape(r, n, h * hd)
    s["q"].copy_(torch.where(live[:, :, None], q, s["q"]))
    s["k"][req, :, at] = rotated(x[:, :, h : h + g], s["k_norm"])[req, tok].to(s["k"].dtype)
    s["v"][req, :, at] = x[req, tok, h + g :].to(s["v"].dtype)
    s["scores"][req, :, at] = 0.0
    s["slot_positions"][req, :, at] = s["positions"][req, tok][:, None].expand(-1, g)
    return {k: s[k] for k in ("q", "k", "v", "scores", "slot_positions")}


def _plain_attend(s):
    c = s["case"]
    r, n, h, g, hd, cap, p = c["requests"], c["tokens"], c["heads"], c["kv_heads"], c["hd"], c["cap"], c["prefix"]
    rep = h // g
    q = s["q"].view(r, n, g, rep, hd).permute(0, 2, 1, 3, 4).reshape(r, g, n * rep, hd) * hd**-0.5
    score = q @ s["k"].float().transpose(2, 3).contiguous()
    last = s["lens"][:, None] - s["new"][:, None] + torch.arange(n, device="cuda")  # the token's own slot
    seen = (torch.arange(cap, device="cuda") <= last[:, :, None]).repeat_interleave(rep, 1)[:, None]
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    if p:
        shared = q.transpose(0, 1).reshape(g, r * n * rep, hd) @ s["prefix_k"].float().transpose(1, 2).contiguous()
        score = torch.cat((shared.view(g, r, n * rep, p).transpose(0, 1), score), 3)
    top = score.amax(3, keepdim=True)
    weight = torch.exp(score - top)
    weight = weight / weight.sum(3, keepdim=True)
    res = weight[..., p:] @ s["v"].float()
    if p:
        shared = weight[..., :p].transpose(0, 1).reshape(g, r * n * rep, p) @ s["prefix_v"].float()
        res = res + shared.view(g, r, n * rep, hd).transpose(0, 1)
    res = res.view(r, g, n, rep, hd).permute(0, 2, 1, 3, 4).reshape(r, n, h * hd)
    live = torch.arange(n, device="cuda") < s["new"][:, None]
    out = torch.where(live[:, :, None], res, s["out"])
    if c["op"] == "attend":
        return out
    weight = torch.where(live.repeat_interleave(rep, 1)[:, None, :, None], weight, torch.zeros_like(weight))
    total = weight.sum(2)
    used = (torch.arange(cap, device="cuda") < s["lens"][:, None])[:, None]
    res = {"out": out, "weights_out": torch.where(used, s["weights"] + total[..., p:], s["weights_out"])}
    if p:
        res["prefix_weights_out"] = s["prefix_weights"] + total[..., :p].sum(0)
    return res


def _plain_evict(s):
    c = s["case"]
    cap, g = c["cap"], c["kv_heads"]
    n = s["lens"].repeat(c["layers"])[:, None, None]
    left = n.clamp(max=c["keep"])
    slot = torch.arange(cap, device="cuda").expand(s["scores"].shape)
    used = slot < n
    pos = s["positions"]
    newest = torch.where(used, pos, torch.full_like(pos, -1)).amax(2, keepdim=True)
    kind = used.int() + (used & ((pos > newest - c["recent"]) | (pos < c["sinks"]))).int()
    order = torch.sort(s["scores"], dim=2, descending=True, stable=True).indices
    order = order.gather(2, torch.sort(kind.gather(2, order), dim=2, descending=True, stable=True).indices)
    rank = torch.empty_like(order).scatter_(2, order, slot)
    kept = rank < left
    hole, mover = (slot < left) & ~kept, (slot >= left) & kept
    movers = torch.sort((~mover).int(), dim=2, stable=True).indices
    come = torch.where(hole, movers.gather(2, (hole.cumsum(2) - 1).clamp(min=0)), slot)
    a, b, to = hole.nonzero(as_tuple=True)
    at = come[a, b, to]
    s["k"][a, b, to] = s["k"][a, b, at]
    s["v"][a, b, to] = s["v"][a, b, at]
    stays = slot < left
    return {"k": s["k"], "v": s["v"], "scores_out": torch.where(stays, s["scores"].gather(2, come), s["scores_out"]),
            "positions_out": torch.where(stays, pos.gather(2, come), s["positions_out"]), "lens_out": s["lens"].clamp(max=c["keep"])}


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attend": _plain_attend, "weigh": _plain_attend, "evict": _plain_evict}[state["case"]["op"]](state)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    new, used = _ragged(case)
    g, hd = case["kv_heads"], case["hd"]
    e = 2 if case["type"] == "f16" else 4
    row = g * hd * e  # one token's keys (or values) in the cache
    if case["op"] == "evict":
        nbytes = 0.0
        for n in used:
            keep, tail = min(n, case["keep"]), max(0, n - case["keep"])
            fixed = min(case["recent"], n) + min(case["sinks"], n)
            free = max(0, keep - fixed)  # chosen by score, anywhere among the rest
            if case["shuffled"]:
                moved = keep * tail / n
            else:
                late = min(case["recent"], tail)
                moved = late + free * (tail - late) / max(1, n - fixed)
            nbytes += case["layers"] * (4 * row * moved + g * (8 * n + 8 * keep))
        return {"bytes": nbytes, "flops": 0.0}
    h = case["heads"]
    tokens = sum(new)
    if case["op"] == "append":
        return {"bytes": tokens * (4 * (2 * h + 2 * g) * hd + 2 * row + 8 * g), "flops": tokens * (h + g) * hd * 8.0}
    p = case["prefix"]
    seen = sum(t * p + t * u - t * (t - 1) // 2 for t, u in zip(new, used))
    nbytes = 2 * row * (p + sum(used)) + 8 * h * hd * tokens
    if case["op"] == "weigh":
        nbytes += 8 * g * (p + sum(used))
    return {"bytes": nbytes, "flops": 4.0 * h * hd * seen}


# --------------------------------------------------------------------------
# the same in 64 bits, request by request and head by head
# --------------------------------------------------------------------------
def _exact_append(case, s):
    r, n, h, g, hd = case["requests"], case["tokens"], case["heads"], case["kv_heads"], case["hd"]
    new, used = _ragged(case)
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    scores, where = s["scores"].double(), s["slot_positions"].clone()
    turn = torch.exp(-math.log(ROPE_BASE) * torch.arange(hd // 2, dtype=torch.float64, device="cuda") / (hd // 2))
    for b in range(r):
        x = s["qkv"][b, : new[b]].double().reshape(new[b], h + 2 * g, hd)
        lo, hi = used[b] - new[b], used[b]
        phase = torch.polar(torch.ones(new[b], hd // 2, dtype=torch.float64, device="cuda"), s["positions"][b, : new[b], None].double() * turn)

        def head(y, gain):
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / hd + EPS) * gain.double()
            z = torch.view_as_complex(y.reshape(new[b], -1, hd // 2, 2).contiguous()) * phase[:, None]
            return torch.view_as_real(z).reshape(y.shape)

        q[b, : new[b]] = head(x[:, :h], s["q_norm"]).reshape(new[b], h * hd)
        k[b, :, lo:hi] = head(x[:, h : h + g], s["k_norm"]).transpose(0, 1)
        v[b, :, lo:hi] = x[:, h + g :].transpose(0, 1)
        scores[b, :, lo:hi] = 0.0
        where[b, :, lo:hi] = s["positions"][b, : new[b]]
    return {"q": q, "k": k, "v": v, "scores": scores, "slot_positions": where}


def _exact_attend(case, s):
    r, n, h, g, hd, p = (case[x] for x in ("requests", "tokens", "heads", "kv_heads", "hd", "prefix"))
    rep = h // g
    new, used = _ragged(case)
    out = s["out"].double()
    if case["op"] == "weigh":
        wo = s["weights_out"].double()
        wp = s["prefix_weights"].double() if p else None
    for b in range(r):
        t, u = new[b], used[b]
        for j in range(g):
            keys, values = s["k"][b, j, :u].double(), s["v"][b, j, :u].double()
            if p:
                keys, values = torch.cat((s["prefix_k"][j].double(), keys)), torch.cat((s["prefix_v"][j].double(), values))
            q = s["q"][b, :t].double().reshape(t, h, hd)[:, j * rep : (j + 1) * rep]
            x = (q.reshape(t * rep, hd) @ keys.t() / math.sqrt(hd)).reshape(t, rep, p + u)
            unseen = torch.ones(t, p + u, dtype=torch.bool, device="cuda").triu(p + u - t + 1)
            x.masked_fill_(unseen[:, None], -math.inf)
            x = torch.exp(x - torch.logsumexp(x, 2, keepdim=True))
            out[b, :t].view(t, h, hd)[:, j * rep : (j + 1) * rep] = (x.reshape(t * rep, p + u) @ values).reshape(t, rep, hd)
            if case["op"] == "weigh":
                total = x.sum((0, 1))
                wo[b, j, :u] = s["weights"][b, j, :u].double() + total[p:]
                if p:
                    wp[j] += total[:p]
    if case["op"] == "attend":
        return out
    res = {"out": out, "weights_out": wo}
    if p:
        res["prefix_weights_out"] = wp
    return res


def _exact_evict(case, s):
    layers, r, g = case["layers"], case["requests"], case["kv_heads"]
    _, used = _ragged(case)
    pos, score = s["positions"].cpu().numpy(), s["scores"].double().cpu().numpy()
    pos_out, score_out = s["positions_out"].cpu().numpy().copy(), s["scores_out"].double().cpu().numpy().copy()
    at, to = [], []
    for i in range(layers * r):
        n = used[i % r]
        m = min(n, case["keep"])
        for j in range(g):
            p, x = pos[i, j, :n], score[i, j, :n]
            safe = (p > p.max() - case["recent"]) | (p < case["sinks"])
            best = np.lexsort((np.arange(n), -x, ~safe))[:m]  # safe ones first, then heavy ones, then low slots
            kept = np.zeros(n, bool)
            kept[best] = True
            holes, movers = np.flatnonzero(~kept[:m]), m + np.flatnonzero(kept[m:])
            come = np.arange(m)
            come[holes] = movers
            pos_out[i, j, :m], score_out[i, j, :m] = p[come], x[come]
            base = (i * g + j) * case["cap"]
            at.append(base + movers)
            to.append(base + holes)
    at, to = (torch.from_numpy(np.concatenate(x)).cuda() for x in (at, to))
    res = {"scores_out": torch.from_numpy(score_out), "positions_out": torch.from_numpy(pos_out),
           "lens_out": torch.tensor([min(n, case["keep"]) for n in used], dtype=torch.int32)}
    for name in ("k", "v"):  # moved, not computed: their own type
        x = s[name].clone().view(-1, case["hd"])
        x[to] = x[at]
        res[name] = x.view(s[name].shape)
    return res


def exact(case, seed):
    s = _inputs(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "weigh": _exact_attend, "evict": _exact_evict}[case["op"]](case, s)
