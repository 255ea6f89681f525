"""Timed cases of the paged 4-bit KV cache (``s2hip.PagedKv``): what a program that
serves many sessions out of one pool of pages calls.

* ``append``  -- head norms, rotation (interleaved or half layout, part of the head,
  scaled frequencies) of the new tokens, keys and values written to their pages in 4
  bits; the values that the cache then holds come back too.
* ``attend``  -- attention of the new tokens over the requests' pages.
* ``update``  -- the requests' page lists made anew: forked, cut, freed and grown; a
  shared page that is about to be written gets a copy in every layer.
* ``compact`` -- the pages in use moved to the front of the pool, in every layer.

With ``own`` false, ``run`` computes them from elementary torch operations in float32
(what is rounded to 4 bits, and angles, in float64); with ``own`` true it calls the
framework.

A page holds ``page`` tokens of every kv head.  A kv head's part of it: codes of the
keys, codes of the values, scales of the keys, scales of the values.  32 elements of a
head share a scale d (float16): an element is d (code - 8).
"""

import math
import os
import sys

import numpy as np
import torch

own = False

ROPE_BASE = 1.0e6
EPS = 1.0e-6


def listed():
    return [
        # a decode step of eight sessions: launch latency
        {"name": "append_step_8", "op": "append", "requests": 8, "tokens": 1, "slots": 2012, "page": 64, "heads": 32, "kv_heads": 8, "hd": 128, "half": False, "rope_dims": 128, "scaling": "none", "factor": 1.0},
        # eight sessions bring a turn of text each, half layout, far positions of a stretched context
        {"name": "append_turn_8", "op": "append", "requests": 8, "tokens": 250, "slots": 1750, "page": 64, "heads": 32, "kv_heads": 8, "hd": 128, "half": True, "rope_dims": 128, "scaling": "parts", "factor": 8.0},
        # an odd turn of three on the small model's heads, a quarter of the head rotated, pages of 16
        {"name": "append_part_3", "op": "append", "requests": 3, "tokens": 37, "slots": 131, "page": 16, "heads": 8, "kv_heads": 2, "hd": 64, "half": False, "rope_dims": 16, "scaling": "linear", "factor": 4.0},
        # three short sessions of the small model: launch latency
        {"name": "attend_step_3", "op": "attend", "requests": 3, "tokens": 1, "shared": 100, "slots": 20, "page": 16, "heads": 8, "kv_heads": 2, "hd": 64},
        # eight voice-clone sessions that were forked from one 1500-token prompt, one decode step
        {"name": "attend_step_8", "op": "attend", "requests": 8, "tokens": 1, "shared": 1500, "slots": 512, "page": 64, "heads": 32, "kv_heads": 8, "hd": 128},
        # sixteen long sessions that share nothing
        {"name": "attend_step_16_long", "op": "attend", "requests": 16, "tokens": 1, "shared": 0, "slots": 32001, "page": 64, "heads": 32, "kv_heads": 8, "hd": 128},
        # eight sessions bring a turn of text each (ragged) over their prompt
        {"name": "attend_turn_8", "op": "attend", "requests": 8, "tokens": 250, "shared": 1500, "slots": 250, "page": 64, "heads": 32, "kv_heads": 8, "hd": 128},
        # a long prompt sees itself
        {"name": "attend_prompt", "op": "attend", "requests": 1, "tokens": 3999, "shared": 0, "slots": 3999, "page": 128, "heads": 32, "kv_heads": 8, "hd": 128},
        # sixteen sessions: some end, some are forked anew from the prompt, all grow by a token
        {"name": "update_16", "op": "update", "requests": 16, "layers": 4, "shared": 1500, "slots": 700, "page": 64, "kv_heads": 8, "hd": 128, "grow": 1},
        # the beams of eight sessions are sorted anew, every layer of their last pages copied
        {"name": "update_64_layers", "op": "update", "requests": 64, "layers": 36, "shared": 6001, "slots": 501, "page": 64, "kv_heads": 8, "hd": 128, "grow": 3},
        # one layer of a small pool
        {"name": "compact_1", "op": "compact", "requests": 8, "layers": 1, "slots": 2001, "page": 32, "kv_heads": 8, "hd": 128, "holes": 0.4},
        # every layer of a pool in which half of the sessions have ended
        {"name": "compact_36", "op": "compact", "requests": 12, "layers": 36, "slots": 3500, "page": 64, "kv_heads": 8, "hd": 128, "holes": 0.5},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "append", "update", "compact"])
    heads, kv_heads, hd = rng.choice([(32, 8, 128), (32, 8, 128), (8, 2, 64), (16, 16, 64), (24, 8, 128), (14, 2, 128)])
    c = {"op": op, "requests": _log_int(rng, 1, 16), "page": rng.choice([16, 32, 64, 64, 128]), "kv_heads": kv_heads, "hd": hd}
    if op == "update":
        return dict(c, requests=_log_int(rng, 1, 64), layers=rng.choice([1, 4, 18]), shared=rng.choice([0, _log_int(rng, 1, 6000)]),
                    slots=_log_int(rng, 1, 600), grow=rng.choice([1, 1, _log_int(rng, 2, 300)]))
    if op == "compact":
        return dict(c, layers=rng.choice([1, 1, 4]), slots=_log_int(rng, 20, 6000), holes=round(rng.uniform(0.1, 0.7), 2))
    c["heads"] = heads
    if rng.random() < 0.5:
        c["tokens"] = rng.choice([1, 1, 2, 3, 4])
        c["slots"] = c["tokens"] - 1 + _log_int(rng, 1, 6000)
    else:
        c["requests"] = min(c["requests"], 8)
        c["tokens"] = _log_int(rng, 5, 2000 // c["requests"])
        c["slots"] = c["tokens"] + rng.choice([0, 0, _log_int(rng, 1, 500)])
    if op == "append":
        return dict(c, half=rng.random() < 0.5, rope_dims=rng.choice([hd, hd, hd // 2, 16]), scaling=rng.choice(["none", "linear", "stretch", "parts"]),
                    factor=rng.choice([2.0, 4.0, 8.0]))
    c["shared"] = rng.choice([0, _log_int(rng, 1, 6000)])
    if c["tokens"] > 4:
        c["shared"] = min(c["shared"], 1500)
    return c


def _ragged(case):
    """(new tokens, tokens in use) of each request; the new tokens are the last ones."""
    n, s, r = case.get("tokens", 0), case["slots"], case["requests"]
    new = [n - (b * 29) % (n // 2 + 1) for b in range(r)]
    used = [case.get("shared", 0) + max(new[b], s - b * (s // (2 * r))) for b in range(r)]
    return new, used


def _sources(case):
    """update: (row taken, tokens of it kept, tokens added) of each request."""
    r, used = case["requests"], _ragged(case)[1]
    source, keep, add = [], [], []
    for b in range(r):
        kind = b % 8 if r > 1 else 0
        source.append(b - 1 if kind in (3, 5) else 0 if kind == 6 else b)  # 3, 5: a neighbour's beam; 6: a new session from the prompt
        keep.append(case.get("shared", 0) if kind == 6 else 0 if kind == 4 else used[b] // 2 if kind == 7 else 1 << 20)  # 4: ended; 7: rewound
        add.append(0 if kind == 4 else case["grow"])
    return source, keep, add


# --------------------------------------------------------------------------
# 4-bit pages
# --------------------------------------------------------------------------
def _rounded8(x):
    """x (float64) to 8 significant bits, ties to even, at the bottom to multiples of 2^-24: a float16 number."""
    exponent = torch.frexp(x).exponent.clamp(min=-16)
    return torch.ldexp(torch.round(torch.ldexp(x, 8 - exponent)), exponent - 8)


def _quantised(x):
    """Codes (uint8, like x) and scales (one per 32 elements) of x [..., hd] in float64."""
    y = x.reshape(*x.shape[:-1], -1, 32)
    at = y.abs().argmax(-1, keepdim=True)
    at = torch.where(y.abs() == y.abs().amax(-1, keepdim=True), torch.arange(32, device=x.device), torch.full_like(at, 32)).amin(-1, keepdim=True)
    d = _rounded8(y.gather(-1, at) / -8)
    code = torch.where(d == 0, torch.zeros_like(y), torch.round(y / torch.where(d == 0, torch.ones_like(d), d))).clamp(-8, 7) + 8
    return code.reshape(x.shape).to(torch.uint8), d.squeeze(-1)


def _key_bytes(code):
    """[..., hd] codes of a key as hd / 2 bytes: dims 32 j + 8 i + 0 .. 7 in the 4 bytes of place (i, j)."""
    c = code.reshape(*code.shape[:-1], -1, 4, 8).transpose(-3, -2)
    first, second = c[..., [0, 4, 1, 5]], c[..., [2, 6, 3, 7]]
    return (first | (second << 4)).reshape(*code.shape[:-1], -1)


def _chunk(case):
    """Where a kv head's parts of a page begin: key codes, value codes, key scales, value scales, end."""
    p, hd = case["page"], case["hd"]
    return [0, p * hd // 2, p * hd, p * hd + p * hd // 16, p * hd + p * hd // 8]


def _value_byte(case, slot):
    """Byte of dims 2 i, 2 i + 1 (i = 0 .. hd / 2 - 1) of the value in a page's slot, from the value codes on."""
    i = torch.arange(case["hd"] // 2, device=slot.device)
    group, pair, tile, four, one = i // 16, i % 16, slot // 16, slot % 16 // 4, slot % 4
    groups = case["hd"] // 32
    return (((tile * 4 + four)[..., None] * 16 + pair) * groups + group) * 4 + one[..., None]


def _value_scale(case, slot):
    """Place of group j's scale of the value in a page's slot, among the value scales."""
    groups = case["hd"] // 32
    return ((slot // 16 * 4 + slot % 16 // 4)[..., None] * groups + torch.arange(groups, device=slot.device)) * 4 + (slot % 4)[..., None]


def _pages_of(keys, values, case):
    """Pages of bytes [pages][kv_heads][chunk] that hold keys, values [pages][kv_heads][page][hd]."""
    e = _chunk(case)
    n, g, p, hd = keys.shape
    out = torch.zeros(n, g, e[4], dtype=torch.uint8, device=keys.device)
    slot = torch.arange(p, device=keys.device)
    code, d = _quantised(keys)
    out[:, :, e[0] : e[1]] = _key_bytes(code).flatten(2)
    out[:, :, e[2] : e[3]] = d.to(torch.float16).view(torch.uint8).flatten(2)
    code, d = _quantised(values)
    at = _value_byte(case, slot).flatten()
    out[:, :, e[1] : e[2]].index_copy_(2, at, (code[..., 0::2] | (code[..., 1::2] << 4)).flatten(2))
    place = _value_scale(case, slot).flatten()
    part = torch.zeros(n, g, p * hd // 32, dtype=torch.float16, device=keys.device).index_copy_(2, place, d.to(torch.float16).flatten(2))
    out[:, :, e[3] :] = part.view(torch.uint8)
    return out


def _held(pages, case):
    """Keys and values [..., page, hd] in float32 that pages of bytes [..., chunk] hold."""
    e, p, hd = _chunk(case), case["page"], case["hd"]
    slot = torch.arange(p, device=pages.device)
    b = pages[..., e[0] : e[1]].reshape(*pages.shape[:-1], p, 4, hd // 32, 4)
    code = torch.stack((b[..., 0] & 15, b[..., 2] & 15, b[..., 0] >> 4, b[..., 2] >> 4, b[..., 1] & 15, b[..., 3] & 15, b[..., 1] >> 4, b[..., 3] >> 4), -1)
    d = pages[..., e[2] : e[3]].contiguous().view(torch.float16).float().reshape(*pages.shape[:-1], p, hd // 32, 1)
    keys = (code.transpose(-3, -2).reshape(*pages.shape[:-1], p, hd // 32, 32).float() - 8.0) * d
    b = pages[..., e[1] : e[2]].index_select(-1, _value_byte(case, slot).flatten()).reshape(*pages.shape[:-1], p, hd // 2)
    code = torch.stack((b & 15, b >> 4), -1).reshape(*pages.shape[:-1], p, hd // 32, 32)
    d = pages[..., e[3] :].contiguous().view(torch.float16).index_select(-1, _value_scale(case, slot).flatten()).float()
    values = (code.float() - 8.0) * d.reshape(*pages.shape[:-1], p, hd // 32, 1)
    return keys.flatten(-2), values.flatten(-2)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _inputs(case, seed):
    """The tensors of a case, from its seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 2 + 1)

    def normal(*shape, spread=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(spread)

    def whole(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    r, kv, hd, page = case["requests"], case["kv_heads"], case["hd"], case["page"]
    new, used = _ragged(case)
    grow = case.get("grow", 0)
    width = (max(used) + grow + page - 1) // page + 2
    common = case.get("shared", 0) // page  # full pages of the prompt: one for all
    count = (np.array(used) + page - 1) // page
    first = np.cumsum(count - common) - (count - common)
    total = int(common + (count - common).sum())
    pages = int(total / (1.0 - case["holes"])) + 2 if case["op"] == "compact" else total + r * (2 + grow // page) + 5
    # pages were given and taken back many times: they lie anywhere
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    i = torch.arange(width, device="cuda")
    place = torch.where(i < common, i, common + whole(first)[:, None] + i - common)
    table = torch.where(i < whole(count)[:, None], order[place.clamp(max=pages - 1).long()], torch.full_like(order[:1], -1))
    s = {"lens": whole(used), "table": table.contiguous(), "pages": pages, "width": width}
    if case["op"] in ("update", "compact"):
        layers, size = case["layers"], kv * _chunk(case)[4]
        s["pool"] = torch.randint(-(1 << 31), (1 << 31) - 1, (layers, pages, size // 4), generator=g, device="cuda", dtype=torch.int32)
        held = torch.zeros(pages, dtype=torch.int32, device="cuda")
        live = (table >= 0).flatten()
        s["refs"] = held.index_add_(0, table.clamp(min=0).flatten().long(), live.int())
        s["refs_out"] = torch.zeros_like(s["refs"])
        s["table_out"] = torch.full_like(s["table"], -1)
        if case["op"] == "update":
            s["source"], s["keep"], s["add"] = (whole(x) for x in _sources(case))
            s["lens_out"] = torch.zeros_like(s["lens"])
        else:
            s["used_out"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        return s
    n, h = case["tokens"], case["heads"]
    s["new"] = whole(new)
    if case["op"] == "append":
        s["pool"] = torch.zeros(pages, kv, _chunk(case)[4], dtype=torch.uint8, device="cuda")
        s["qkv"] = normal(r, n, (h + 2 * kv) * hd, spread=3.0)
        s["q_norm"] = normal(hd, spread=0.2).add_(1.0)
        s["k_norm"] = normal(hd, spread=0.2).add_(1.0)
        start = torch.randint(0, 60000, (r, 1), generator=g, device="cuda")
        s["positions"] = (start + torch.arange(n, device="cuda")).to(torch.int32)
        s["q"] = torch.zeros(r, n, h * hd, device="cuda")
        s["k_held"] = torch.zeros(r, n, kv * hd, device="cuda")
        s["v_held"] = torch.zeros(r, n, kv * hd, device="cuda")
        return s
    # normed and rotated keys, queries a little larger: scores spread by about 1.5
    s["pool"] = _pages_of(normal(pages, kv, page, hd).double() if pages * kv * page * hd < 1 << 26 else normal(pages, kv, page, hd), normal(pages, kv, page, hd), case)
    s["q"] = normal(r, n, h * hd, spread=1.5)
    s["out"] = torch.zeros(r, n, h * hd, device="cuda")
    return s


_opened = {}


def _ops(case, state):
    """The handle of this model and pool: a program keeps it as long as both."""
    key = tuple(case.get(k, 0) for k in ("heads", "kv_heads", "hd", "page", "half", "rope_dims", "scaling", "factor")) + (state["pages"], state["width"])
    if key not in _opened:
        sys.path.insert(0, os.path.abspath("fish-s2pro_amd"))
        from s2hip import PagedKv, rope_frequencies

        freq, gain = rope_frequencies(case.get("rope_dims", case["hd"]), ROPE_BASE, case.get("scaling", "none"), case.get("factor", 1.0), context=8192)
        _opened[key] = PagedKv(case.get("heads", case["kv_heads"]), case["kv_heads"], case["hd"], page_tokens=case["page"], pages=state["pages"],
                               table_pages=state["width"], max_requests=64, max_tokens=4096, rope_freq=freq, rope_gain=gain, rope_half=case.get("half", False), eps=EPS)
    return _opened[key]


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:  # the handle and where the requests' pages are, which a program keeps per layer
        ops = state["ops"] = _ops(case, state)
        at = lambda name: state[name].data_ptr() if name in state else 0  # noqa: E731
        state["view"] = ops.view(at("pool"), at("table"), at("lens"), case["requests"], new_lens=at("new"))
    return state


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def _run_own(s):
    c, ops, view = s["case"], s["ops"], s["view"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "append":
        ops.append(view, s["qkv"].data_ptr(), c["tokens"], s["positions"].data_ptr(), s["q"].data_ptr(), q_norm=s["q_norm"].data_ptr(),
                   k_norm=s["k_norm"].data_ptr(), k_held=s["k_held"].data_ptr(), v_held=s["v_held"].data_ptr(), stream=stream)
        return {k: s[k] for k in ("q", "k_held", "v_held", "pool")}
    if c["op"] == "attend":
        ops.attend(view, s["q"].data_ptr(), c["tokens"], s["out"].data_ptr(), stream=stream)
        return s["out"]
    if c["op"] == "update":
        ops.update(view, s["refs"].data_ptr(), s["refs_out"].data_ptr(), s["table_out"].data_ptr(), s["lens_out"].data_ptr(), source=s["source"].data_ptr(),
                   keep=s["keep"].data_ptr(), add=s["add"].data_ptr(), layers=c["layers"], stream=stream)
        return {k: s[k] for k in ("pool", "refs_out", "table_out", "lens_out")}
    ops.compact(view, s["refs"].data_ptr(), s["refs_out"].data_ptr(), s["table_out"].data_ptr(), s["used_out"].data_ptr(), layers=c["layers"], stream=stream)
    return {k: s[k] for k in ("pool", "refs_out", "table_out", "used_out")}


def _frequencies(case):
    """Angles per position of each pair, and what cos and sin are multiplied by."""
    dims, factor, base = case["rope_dims"], case["factor"], ROPE_BASE
    if case["scaling"] == "stretch":
        base = base * factor ** (dims / (dims - 2))
    freq = base ** (-torch.arange(0, dims, 2, device="cuda", dtype=torch.float64) / dims)
    if case["scaling"] == "linear":
        return freq / factor, 1.0
    if case["scaling"] == "parts":  # pairs that turn often within the old context stay, slow ones are stretched
        share = ((8192 / (2 * math.pi) * freq - 1.0) / 31.0).clamp(0.0, 1.0)
        return freq / factor * (1.0 - share) + freq * share, 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _plain_append(s):
    c = s["case"]
    r, n, h, g, hd, page = c["requests"], c["tokens"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    x = s["qkv"].view(r, n, h + 2 * g, hd).double()
    freq, gain_ = _frequencies(c)
    angle = s["positions"].double()[:, :, None, None] * freq
    cos, sin = torch.cos(angle) * gain_, torch.sin(angle) * gain_

    def rotated(x, gain):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain.double()
        turn, rest = x[..., : c["rope_dims"]], x[..., c["rope_dims"] :]
        if c["half"]:
            a, b = turn.chunk(2, -1)
            return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)
        a, b = turn[..., 0::2], turn[..., 1::2]
        return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), rest), -1)

    live = torch.arange(n, device="cuda") < s["new"][:, None]
    slot = (s["lens"] - s["new"])[:, None] + torch.arange(n, device="cuda")
    req, tok = live.nonzero(as_tuple=True)
    at = slot[req, tok].long()
    q = rotated(x[:, :, :h], s["q_norm"]).reshape(r, n, h * hd).float()
    s["q"].copy_(torch.where(live[:, :, None], q, s["q"]))
    where = s["table"][req, at // page].long()[:, None, None]
    head = torch.arange(g, device="cuda")[:, None]
    at = at % page
    e = _chunk(c)
    code, d = _quantised(rotated(x[:, :, h : h + g], s["k_norm"])[req, tok])
    row = e[0] + at[:, None] * (hd // 2) + torch.arange(hd // 2, device="cuda")
    s["pool"][where, head, row[:, None]] = _key_bytes(code)
    row = e[2] + at[:, None] * (hd // 16) + torch.arange(hd // 16, device="cuda")
    s["pool"][where, head, row[:, None]] = d.to(torch.float16).view(torch.uint8)
    s["k_held"][req, tok] = ((code.double() - 8) * d.repeat_interleave(32, -1)).float().flatten(1)
    code, d = _quantised(x[req, tok, h + g :])
    s["pool"][where, head, e[1] + _value_byte(c, at)[:, None]] = code[..., 0::2] | (code[..., 1::2] << 4)
    row = (e[3] + 2 * _value_scale(c, at)[..., None] + torch.arange(2, device="cuda")).flatten(1)
    s["pool"][where, head, row[:, None]] = d.to(torch.float16).view(torch.uint8)
    s["v_held"][req, tok] = ((code.double() - 8) * d.repeat_interleave(32, -1)).float().flatten(1)
    return {k: s[k] for k in ("q", "k_held", "v_held", "pool")}


def _plain_attend(s):
    c = s["case"]
    r, n, h, g, hd = c["requests"], c["tokens"], c["heads"], c["kv_heads"], c["hd"]
    rep, width = h // g, s["width"]
    cap = width * c["page"]
    k, v = _held(s["pool"][s["table"].clamp(min=0).flatten().long()].view(r, width, g, -1).transpose(1, 2), c)
    k, v = k.reshape(r, g, cap, hd), v.reshape(r, g, cap, hd)
    q = s["q"].view(r, n, g, rep, hd).permute(0, 2, 1, 3, 4).reshape(r, g, n * rep, hd) * hd**-0.5
    score = q @ k.transpose(2, 3).contiguous()
    last = s["lens"][:, None] - s["new"][:, None] + torch.arange(n, device="cuda")  # the token's own slot
    seen = (torch.arange(cap, device="cuda") <= last[:, :, None]).repeat_interleave(rep, 1)[:, None]
    score = torch.where(seen, score, torch.full_like(score[:1, :1, :1, :1], -math.inf))
    weight = torch.exp(score - score.amax(3, keepdim=True))
    weight = weight / weight.sum(3, keepdim=True)
    res = (weight @ v).view(r, g, n, rep, hd).permute(0, 2, 1, 3, 4).reshape(r, n, h * hd)
    live = torch.arange(n, device="cuda") < s["new"][:, None]
    return torch.where(live[:, :, None], res, s["out"])


def _plain_update(s):
    page, width = s["case"]["page"], s["width"]
    i = torch.arange(width, device="cuda")

    def held(refs, table, used, sign):
        return refs.index_add(0, table.clamp(min=0).flatten().long(), sign * used.flatten().int())

    def pages_of(n):
        return (n + page - 1) // page

    row = s["source"].long()
    kept = torch.minimum(s["keep"], s["lens"][row])
    base = s["table"][row]
    refs = held(held(s["refs"], s["table"], i < pages_of(s["lens"])[:, None], -1), base, i < pages_of(kept)[:, None], 1)
    # the last page of a row that grows, held by others too: all but its last writer write to a copy
    last = base.gather(1, (kept // page).clamp(max=width - 1).long()[:, None]).squeeze(1)
    grows = (kept % page != 0) & (s["add"] > 0)
    order = torch.arange(len(row), device="cuda")
    before = ((last[:, None] == last) & grows & (order[:, None] > order)).sum(1)
    copy = grows & (before < refs[last.clamp(min=0).long()] - 1)
    new_lens = kept + s["add"]
    first = pages_of(kept) - copy.int()
    need = pages_of(new_lens) - first
    free = torch.sort((refs > 0).int(), stable=True).indices.int()
    which = (torch.cumsum(need, 0) - need - first)[:, None] + i
    takes = (i >= first[:, None]) & (i < pages_of(new_lens)[:, None])
    given = free[which.clamp(0, len(refs) - 1).long()]
    table = torch.where(takes, given, torch.where(i < first[:, None], base, torch.full_like(base, -1)))
    refs = held(refs, table, takes, 1).index_add(0, last.clamp(min=0).long(), -copy.int())
    to = table.gather(1, first.clamp(max=width - 1).long()[:, None]).squeeze(1)[copy].long()
    s["pool"][:, to] = s["pool"][:, last[copy].long()]
    return {"pool": s["pool"], "refs_out": refs, "table_out": table, "lens_out": new_lens}


def _plain_compact(s):
    page, refs, table = s["case"]["page"], s["refs"], s["table"]
    ids = torch.arange(len(refs), device="cuda")
    used = (refs > 0).sum()
    mover, hole = (refs > 0) & (ids >= used), (refs == 0) & (ids < used)
    src, dst = mover.nonzero().squeeze(1), hole.nonzero().squeeze(1)
    to = ids.index_put((src,), dst)
    come = ids.index_put((dst,), src)
    live = torch.arange(table.shape[1], device="cuda") < ((s["lens"] + page - 1) // page)[:, None]
    s["pool"][:, dst] = s["pool"][:, src]
    return {"pool": s["pool"], "refs_out": torch.where(ids < used, refs[come], torch.zeros_like(refs)),
            "table_out": torch.where(live, to[table.clamp(min=0).long()].int(), s["table_out"]), "used_out": used.int().view(1)}


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attend": _plain_attend, "update": _plain_update, "compact": _plain_compact}[state["case"]["op"]](state)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def _new_rows(case):
    """update, row by row: (tokens kept, tokens in all) and the pages that are copied."""
    _, used = _ragged(case)
    source, keep, add = _sources(case)
    page, common = case["page"], case.get("shared", 0) // case["page"]
    kept = [min(keep[b], used[source[b]]) for b in range(len(used))]
    name = lambda b, i: ("all", i) if i < common else (b, i)  # noqa: E731
    refs = {}
    for b, k in enumerate(kept):
        for i in range((k + page - 1) // page):
            refs[name(source[b], i)] = refs.get(name(source[b], i), 0) + 1
    copies = 0
    for b, k in enumerate(kept):
        at = name(source[b], k // page)
        if add[b] and k % page and refs[at] > 1:
            refs[at] -= 1
            copies += 1
    return [(k, k + a) for k, a in zip(kept, add)], copies


def work(case):
    new, used = _ragged(case)
    g, hd, page = case["kv_heads"], case["hd"], case["page"]
    row = g * hd * 9 // 8  # one token in the cache
    if case["op"] == "update":
        rows, copies = _new_rows(case)
        lists = sum((u + page - 1) // page for u in used) + sum((n + page - 1) // page for _, n in rows)
        return {"bytes": 4.0 * lists + 2.0 * copies * case["layers"] * page * row, "flops": 0.0}
    if case["op"] == "compact":
        pages = sum((u + page - 1) // page for u in used)
        return {"bytes": 8.0 * pages + 2.0 * pages * case["holes"] * case["layers"] * page * row, "flops": 0.0}
    h, tokens = case["heads"], sum(new)
    if case["op"] == "append":
        return {"bytes": tokens * (4.0 * (2 * h + 4 * g) * hd + row), "flops": tokens * (h + g) * hd * 8.0}
    shared = case["shared"] // page * page
    seen = sum(t * u - t * (t - 1) // 2 for t, u in zip(new, used))
    return {"bytes": row * (shared + sum(u - shared for u in used)) + 8.0 * h * hd * tokens, "flops": 4.0 * h * hd * seen}


# --------------------------------------------------------------------------
# the same in 64 bits, request by request and head by head
# --------------------------------------------------------------------------
def _exact_held(x):
    """What 4 bits hold of x [..., hd] (float64)."""
    y = x.reshape(-1, 32)
    big, at = y.abs().max(1)
    low = torch.where(y.abs() == big[:, None], torch.arange(32, device=x.device), torch.full_like(at, 99)[:, None]).min(1).values
    d = y[torch.arange(len(y), device=x.device), low] / -8
    unit = 2.0 ** torch.clamp(torch.floor(torch.log2(d.abs().clamp(min=2.0**-60))) - 7, min=-24)
    d = torch.round(d / unit) * unit
    steps = torch.clamp(torch.round(y / d[:, None]), -8, 7)
    return torch.where(d[:, None] == 0, torch.zeros_like(y), steps * d[:, None]).reshape(x.shape)


def _exact_append(case, s):
    n, h, g, hd, dims = case["tokens"], case["heads"], case["kv_heads"], case["hd"], case["rope_dims"]
    new, _ = _ragged(case)
    res = {k: s[k].double() for k in ("q", "k_held", "v_held")}
    f, factor = [], case["factor"]
    for i in range(dims // 2):
        w = math.exp(-2.0 * i / dims * (math.log(ROPE_BASE) + (dims / (dims - 2.0) * math.log(factor) if case["scaling"] == "stretch" else 0.0)))
        if case["scaling"] == "linear":
            w /= factor
        if case["scaling"] == "parts":
            fast = min(1.0, max(0.0, (8192 * w / (2 * math.pi) - 1.0) / (32.0 - 1.0)))
            w = fast * w + (1.0 - fast) * w / factor
        f.append(w)
    size = 1.0 + 0.1 * math.log(factor) if case["scaling"] == "parts" else 1.0
    f = torch.tensor(f, dtype=torch.float64, device="cuda")
    even = torch.arange(dims // 2, device="cuda") * (1 if case["half"] else 2)
    odd = even + (dims // 2 if case["half"] else 1)
    for b in range(case["requests"]):
        t = new[b]
        x = s["qkv"][b, :t].double().reshape(t, h + 2 * g, hd)
        phase = torch.polar(torch.full((t, 1, dims // 2), size, dtype=torch.float64, device="cuda"), s["positions"][b, :t, None, None].double() * f)

        def head(y, gain):
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / hd + EPS) * gain.double()
            z = torch.complex(y[..., even], y[..., odd]) * phase
            y[..., even], y[..., odd] = z.real, z.imag
            return y

        res["q"][b, :t] = head(x[:, :h], s["q_norm"]).reshape(t, h * hd)
        res["k_held"][b, :t] = _exact_held(head(x[:, h : h + g], s["k_norm"])).reshape(t, g * hd)
        res["v_held"][b, :t] = _exact_held(x[:, h + g :]).reshape(t, g * hd)
    return dict(res, pool=None)


def _exact_attend(case, s):
    r, h, g, hd, page = (case[x] for x in ("requests", "heads", "kv_heads", "hd", "page"))
    rep, groups = h // g, case["hd"] // 32
    new, used = _ragged(case)
    out = s["out"].double()
    e = _chunk(case)
    low = torch.arange(8, device="cuda") // 2 * 4 + torch.arange(8, device="cuda") % 2 * 16  # bits of a key's eight dims
    for b in range(r):
        t, u = new[b], used[b]
        ids = s["table"][b, : (u + page - 1) // page].long()
        for j in range(g):
            part = s["pool"][ids, j]
            words = part[:, : e[1]].contiguous().view(torch.int32).view(len(ids), page, 4, groups)
            keys = ((words[..., None] >> low) & 15).permute(0, 1, 3, 2, 4).reshape(-1, groups, 32).double() - 8
            keys = (keys * part[:, e[2] : e[3]].contiguous().view(torch.float16).view(-1, groups, 1).double()).view(-1, hd)[:u]
            bytes_ = part[:, e[1] : e[2]].reshape(len(ids), page // 16, 4, 16, groups, 4).permute(0, 1, 2, 5, 4, 3)
            values = torch.stack((bytes_ & 15, bytes_ >> 4), -1).reshape(-1, groups, 32).double() - 8
            d = part[:, e[3] :].contiguous().view(torch.float16).view(len(ids), page // 16, 4, groups, 4).permute(0, 1, 2, 4, 3)
            values = (values * d.reshape(-1, groups, 1).double()).view(-1, hd)[:u]
            q = s["q"][b, :t].double().reshape(t, h, hd)[:, j * rep : (j + 1) * rep]
            x = (q.reshape(t * rep, hd) @ keys.t().contiguous() / math.sqrt(hd)).reshape(t, rep, u)
            x.masked_fill_(torch.ones(t, u, dtype=torch.bool, device="cuda").triu(u - t + 1)[:, None], -math.inf)
            x = torch.exp(x - torch.logsumexp(x, 2, keepdim=True))
            out[b, :t].view(t, h, hd)[:, j * rep : (j + 1) * rep] = (x.reshape(t * rep, u) @ values).reshape(t, rep, hd)
    return out


def _exact_update(case, s):
    page, r, width = case["page"], case["requests"], s["width"]
    _, used = _ragged(case)
    source, keep, add = _sources(case)
    old, refs = s["table"].cpu().numpy(), s["refs"].cpu().numpy().copy()
    count = lambda n: (n + page - 1) // page  # noqa: E731
    table = np.full((r, width), -1, np.int32)
    kept = [min(keep[b], used[source[b]]) for b in range(r)]
    for b in range(r):
        for p in old[b, : count(used[b])]:
            refs[p] -= 1
    for b in range(r):
        table[b, : count(kept[b])] = old[source[b], : count(kept[b])]
        for p in table[b, : count(kept[b])]:
            refs[p] += 1
    free = [p for p in range(len(refs)) if refs[p] == 0][::-1]
    at, to = [], []
    for b in range(r):
        tail = kept[b] // page
        if add[b] and kept[b] % page and refs[table[b, tail]] > 1:
            refs[table[b, tail]] -= 1
            at.append(int(table[b, tail]))
            to.append(free.pop())
            table[b, tail], refs[to[-1]] = to[-1], 1
        for i in range(count(kept[b]), count(kept[b] + add[b])):
            table[b, i] = free.pop()
            refs[table[b, i]] = 1
    pool = s["pool"].clone()
    pool[:, to] = pool[:, at]
    return {"pool": pool, "refs_out": torch.from_numpy(refs), "table_out": torch.from_numpy(table),
            "lens_out": torch.tensor([k + a for k, a in zip(kept, add)], dtype=torch.int32)}


def _exact_compact(case, s):
    refs, table = s["refs"].cpu().numpy(), s["table"].cpu().numpy()
    _, used = _ragged(case)
    n = int((refs > 0).sum())
    holes, movers = np.flatnonzero(refs[:n] == 0), n + np.flatnonzero(refs[n:] > 0)
    to = dict(zip(movers.tolist(), holes.tolist()))
    out, res = s["table_out"].cpu().numpy().copy(), np.zeros_like(refs)
    for b, u in enumerate(used):
        m = (u + case["page"] - 1) // case["page"]
        out[b, :m] = [to.get(p, p) for p in table[b, :m].tolist()]
    for p in np.flatnonzero(refs).tolist():
        res[to.get(p, p)] = refs[p]
    pool = s["pool"].clone()
    pool[:, holes.tolist()] = pool[:, movers.tolist()]
    return {"pool": pool, "refs_out": torch.from_numpy(res), "table_out": torch.from_numpy(out), "used_out": torch.tensor([n], dtype=torch.int32)}


def exact(case, seed):
    s = _inputs(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "update": _exact_update, "compact": _exact_compact}[case["op"]](case, s)
