"""The block-scaled cache: what is measured of it, over which ranges, and its operators in their plain form.

A block-scaled store holds rows of ``hd`` numbers as blocks of 32: 4-bit (E2M1) or 8-bit (E4M3) codes and one
power of two for a block.  ``codes`` is (batch, heads, rows, hd * bits / 8) bytes, column 2 i of a 4-bit row in the
low half of byte i; ``scale`` is (batch, heads, rows, hd / 32) bytes, e standing for 2^(e - 127).  The kinds of a case:

  store   a prompt's keys and values written into a cache, and all of its rows read back
  rows    the rows that a list of ids names read back
  attn    one token's attention over what the cache holds
  step    the same with the token's own row written first: what a layer does at a decode step

A case is a dict of plain values: kind, batch, hkv, group, hd, rows (the longest sequence; the room of the cache),
ragged (sequences of other lengths), kbits, vbits, ids, sink, window (rows attended: the first ``sink`` and the last
``window``; 0: all of them).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
EMAX = {4: 2, 8: 8}                       # exponent of the largest code of a format
MOST = {4: 6.0, 8: 448.0}                 # that code
BUMP = {4: 0x200000, 8: 0x17ffff}         # carries into the exponent where the largest number would round past that code
BYTES = {4: (2, 252), 8: (10, 246)}       # scales for which every number of a block is a normal bf16 number or zero


def _case(name, kind, batch, hkv, hd, rows, group=1, ragged=False, kbits=4, vbits=4, ids=0, sink=0, window=0):
    return dict(name=name, kind=kind, batch=batch, hkv=hkv, group=group, hd=hd, rows=rows, ragged=ragged, kbits=kbits,
                vbits=vbits, ids=ids, sink=sink, window=window)


def listed():
    return [
        # a chat turn's prompt: latency
        _case("store_chat_512", "store", 1, 8, 128, 512),
        # a document of about 32K tokens
        _case("store_doc_32k", "store", 1, 8, 128, 32601),
        # three wide-headed prompts, 8-bit keys and values
        _case("store_wide_3x24k", "store", 3, 4, 256, 24683, kbits=8, vbits=8),
        # the rows that a retrieval step selected, for a harness that attends over a bf16 buffer
        _case("rows_doc_1k", "rows", 1, 8, 128, 32601, ids=1092),
        # the same of a served batch
        _case("rows_serve_2k", "rows", 8, 8, 128, 131072, ids=2117),
        # a token of a chat turn: latency
        _case("attn_chat_517", "attn", 1, 8, 128, 517, group=4),
        # one document of about 32K tokens
        _case("attn_doc_32k", "attn", 1, 8, 128, 32601, group=4),
        # narrow heads in groups of seven, sequences of many lengths, 8-bit keys
        _case("attn_ragged_5x16k", "attn", 5, 4, 64, 16391, group=7, ragged=True, kbits=8),
        # batched serving at 128K tokens
        _case("attn_serve_8x128k", "attn", 8, 8, 128, 131072, group=4),
        # one sequence of a million tokens
        _case("attn_book_1m", "attn", 1, 8, 128, 1048576, group=4),
        # a layer's step of a chat
        _case("step_chat_4k", "step", 1, 8, 128, 4096, group=4),
        # wide heads, sinks and a recent window, 8-bit keys
        _case("step_wide_3x24k", "step", 3, 4, 256, 24683, group=4, ragged=True, kbits=8, sink=4, window=8192),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_LARGEST = 8 * 8 * 131072 * 128   # elements of K of the largest listed attention


def draw(rng):
    kind = rng.choice(["store", "rows", "attn", "attn", "attn", "step", "step"])
    while True:
        c = _case("", kind, _log_int(rng, 1, 16), rng.choice([1, 2, 4, 5, 8]), rng.choice([64, 128, 128, 256]),
                  _log_int(rng, 1, 1 << 20), kbits=rng.choice([4, 4, 8]), vbits=rng.choice([4, 4, 8]))
        del c["name"]
        c["ragged"] = kind in ("attn", "step") and rng.random() < 0.5
        if kind in ("attn", "step"):
            c["group"] = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
            if rng.random() < 0.3:
                c["sink"], c["window"] = rng.choice([0, 1, 4, 64]), _log_int(rng, 1, c["rows"] + 1)
        if kind == "rows":
            c["ids"] = _log_int(rng, 1, min(c["rows"], 8192))
        cost = c["batch"] * c["hkv"] * c["rows"] * c["hd"] * (c["kbits"] + c["vbits"]) // 8
        if cost <= _LARGEST // (8 if kind == "store" else 1):
            return c


# ---- the format ----------------------------------------------------------------------------------------------------

def _encode(x, bits):
    """x (..., hd) -> codes (..., hd * bits / 8) and scale (..., hd / 32), both uint8."""
    x = x.float().unflatten(-1, (-1, 32))
    most = x.abs().amax(-1).view(torch.int32)
    e = (((most + BUMP[bits]) >> 23) - EMAX[bits]).clamp(*BYTES[bits])
    fine = most < 0x7f800000
    y = x * ((254 - e) << 23).view(torch.float32).unsqueeze(-1)   # 2^(127 - e), exactly
    y = torch.where(fine.unsqueeze(-1), y, 0.0).clamp(-MOST[bits], MOST[bits])
    if bits == 8:
        codes = y.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        a = y.abs()
        c = torch.where(a < 2, (2 * a).round(), torch.where(a < 4, a.round() + 2, (a / 2).round() + 4)).to(torch.uint8)
        c = c | (torch.signbit(y).to(torch.uint8) << 3)
        codes = c[..., ::2] | (c[..., 1::2] << 4)
    return codes.flatten(-2), torch.where(fine, e, 255).to(torch.uint8)


def _decode(codes, scale, bits):
    """The numbers that a store holds, (..., hd) fp32."""
    if bits == 8:
        x = codes.view(torch.float8_e4m3fn).float()
    else:
        half = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
        one = torch.cat([half, -half])
        pair = torch.stack([one.repeat(16), one.repeat_interleave(16)], -1)   # (256, 2): low half first
        x = pair[codes.int()].flatten(-2)
    f = (scale.int() << 23).view(torch.float32)                   # 2^(scale - 127), exactly
    f = torch.where(scale == 255, torch.nan, f)
    return x.unflatten(-1, (-1, 32)).mul_(f.unsqueeze(-1)).flatten(-2)


# ---- the cases ------------------------------------------------------------------------------------------------------

def _keys(shape, g):
    """Keys with channels of unequal size (log-normal), as keys have them; the last dimension is the channel."""
    k = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
    return k.mul_(torch.exp(torch.randn(shape[-1:], generator=g, device=DEV)).to(torch.bfloat16))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    b, h, n, hd, kind = case["batch"], case["hkv"], case["rows"], case["hd"], case["kind"]
    st = {"case": case, "scale": 1.0 / math.sqrt(hd)}
    if kind == "store":     # what a model's projections leave: (batch, tokens, heads, hd); and a cache with room for it
        st["k_src"], st["v_src"] = _keys((b, n, h, hd), g), torch.randn((b, n, h, hd), generator=g, device=DEV, dtype=torch.bfloat16)
        for t, bits in (("k", case["kbits"]), ("v", case["vbits"])):
            st[t] = (torch.zeros((b, h, n, hd * bits // 8), dtype=torch.uint8, device=DEV),
                     torch.zeros((b, h, n, hd // 32), dtype=torch.uint8, device=DEV))
    else:                   # a cache that holds such rows
        room = n + (1 if kind == "step" else 0)
        for t, bits in (("k", case["kbits"]), ("v", case["vbits"])):
            codes = torch.empty((b, h, room, hd * bits // 8), dtype=torch.uint8, device=DEV)
            scale = torch.empty((b, h, room, hd // 32), dtype=torch.uint8, device=DEV)
            for i in range(b):
                for lo in range(0, room, 1 << 17):
                    at = (h, min(room - lo, 1 << 17), hd)
                    x = _keys(at, g) if t == "k" else torch.randn(at, generator=g, device=DEV, dtype=torch.bfloat16)
                    codes[i, :, lo:lo + at[1]], scale[i, :, lo:lo + at[1]] = _encode(x, bits)
            st[t] = (codes, scale)
    if kind == "rows":
        at = torch.rand((b * h, n), generator=g, device=DEV)
        st["idx"] = at.topk(case["ids"], dim=-1).indices.to(torch.int32)
    if kind in ("attn", "step"):
        # (channels are of unequal size, so the logits of such queries are already peaked)
        st["q"] = torch.randn((b, h * case["group"], hd), generator=g, device=DEV, dtype=torch.bfloat16)
        lens = torch.full((b,), n, dtype=torch.int32, device=DEV)
        if case["ragged"]:
            lens = (torch.rand((b,), generator=g, device=DEV) * n).to(torch.int32) + 1
            lens[b // 2] = n
        st["lens"] = lens
    if kind == "step":
        st["new_k"] = _keys((b, h, hd), g)
        st["new_v"] = torch.randn((b, h, hd), generator=g, device=DEV, dtype=torch.bfloat16)
        st["idx"] = lens.view(b, 1).expand(b, h).reshape(b * h, 1).contiguous()
    return st


def _attend(q, k, v, lens, case, scale):
    """q (b, heads, hd) over k, v (b, hkv, rows, hd) in fp32: out in q's type, and the log of the sum of exponentials."""
    b, h, n, hd = k.shape
    s = torch.matmul(q.float().view(b, h, -1, hd), k.transpose(-1, -2)).mul_(scale)
    at = torch.arange(n, device=q.device)
    live = at < lens.view(b, 1)
    if case["window"]:
        live &= (at < case["sink"]) | (at >= lens.view(b, 1) - case["window"])
    s.masked_fill_(~live.view(b, 1, 1, n), -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    return out.to(q.dtype).view(b, -1, hd), (m + total.log()).view(b, -1)


def run(state):
    case = state["case"]
    kind, b, h, n, hd = case["kind"], case["batch"], case["hkv"], case["rows"], case["hd"]
    if own:
        from diffcache_amd import _hip as hip
        k, v = hip.MxStore(*state["k"]), hip.MxStore(*state["v"])
        if kind == "store":
            hip.mx_ingest(k, v, state["k_src"], state["v_src"])
            return hip.mx_gather_rows(k, v, None, n_idx=n)
        if kind == "rows":
            return hip.mx_gather_rows(k, v, state["idx"])
        if kind == "attn":
            return hip.mx_attn(state["q"], k, v, state["lens"], n_rows=n, n_sink=case["sink"], window=case["window"],
                               want_lse=True)
        out, lse = hip.mx_attn(state["q"], k, v, state["lens"], n_rows=n + 1, n_sink=case["sink"], window=case["window"],
                               new_k=state["new_k"], new_v=state["new_v"], want_lse=True)
        return (out, lse) + hip.mx_gather_rows(k, v, state["idx"])
    if kind == "store":
        for t in ("k", "v"):
            codes, scale = _encode(state[t + "_src"].transpose(1, 2), case[t + "bits"])
            state[t][0].copy_(codes)
            state[t][1].copy_(scale)
        return tuple(_decode(*state[t], case[t + "bits"]).to(torch.bfloat16) for t in ("k", "v"))
    if kind == "rows":
        unit = torch.arange(b * h, device=DEV).unsqueeze(1)
        return tuple(_decode(state[t][0].flatten(0, 1)[unit, state["idx"]], state[t][1].flatten(0, 1)[unit, state["idx"]],
                             case[t + "bits"]).to(torch.bfloat16).view(b, h, -1, hd) for t in ("k", "v"))
    if kind == "attn":
        return _attend(state["q"], _decode(*state["k"], case["kbits"]), _decode(*state["v"], case["vbits"]), state["lens"],
                       case, state["scale"])
    seq, rows = torch.arange(b, device=DEV), []
    for t in ("k", "v"):
        codes, scale = _encode(state["new_" + t], case[t + "bits"])
        state[t][0][seq, :, state["lens"].long()] = codes
        state[t][1][seq, :, state["lens"].long()] = scale
        rows.append(_decode(codes, scale, case[t + "bits"]).to(torch.bfloat16).unsqueeze(2))
    out, lse = _attend(state["q"], _decode(*state["k"], case["kbits"]), _decode(*state["v"], case["vbits"]),
                       state["lens"] + 1, case, state["scale"])
    return out, lse, rows[0], rows[1]


def _attended(case):
    """Rows that one unit attends to, on average."""
    n = case["rows"] * (0.5 * (1 + 1 / case["batch"]) if case["ragged"] else 1)
    return min(n, case["sink"] + case["window"]) if case["window"] else n


def work(case):
    units, hd, kind = case["batch"] * case["hkv"], case["hd"], case["kind"]
    row = hd * (case["kbits"] + case["vbits"]) // 8 + 2 * (hd // 32)   # a token's bytes in the store, K and V
    if kind == "store":     # bf16 in, codes and scales, bf16 out
        return {"bytes": units * case["rows"] * (4 * hd + row + 4 * hd), "flops": units * case["rows"] * 2 * hd * 4}
    if kind == "rows":
        return {"bytes": units * case["ids"] * (4 + row + 4 * hd), "flops": units * case["ids"] * 2 * hd}
    n = _attended(case)
    return {"bytes": int(units * (n * row + 4 * case["group"] * hd + (4 * hd + row if kind == "step" else 0))),
            "flops": int(units * n * case["group"] * 4 * hd)}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _grid(bits):
    """Every number a code of the format stands for, by its code."""
    out = []
    m_bits, e_bits, bias = (1, 2, 1) if bits == 4 else (3, 4, 7)
    for c in range(1 << bits):
        sign, e, m = c >> (bits - 1), (c >> m_bits) & ((1 << e_bits) - 1), c & ((1 << m_bits) - 1)
        x = math.ldexp(m, 1 - bias - m_bits) if e == 0 else math.ldexp(m + (1 << m_bits), e - bias - m_bits)
        if bits == 8 and (c & 127) == 127:
            x = math.nan
        out.append(-x if sign else x)
    return torch.tensor(out, dtype=torch.float64, device=DEV)


def _power(e):
    """2^e in 64 bits, exactly; e whole numbers."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _numbers(codes, scale, bits):
    """The numbers of a piece of a store, in 64 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2) if bits == 4 else codes
    x = _grid(bits).take(c.long())
    return x * _power(scale.long() - 127).masked_fill(scale == 255, math.nan).repeat_interleave(32, -1)


def _rounded(x, bits):
    """x in 64 bits -> the nearest numbers that a block of the format can hold (ties to the even code), with the least
    scale at which the block's largest number does not round past the last code."""
    grid = _grid(bits)[:7 + 1 if bits == 4 else 126 + 1]
    blocks = x.reshape(-1, 32)
    most = blocks.abs().amax(-1)
    beyond = 7.0 if bits == 4 else 464.0                       # half a step past the last code, whose tie ...
    past = (lambda u: u >= beyond) if bits == 4 else (lambda u: u > beyond)   # ... goes up (odd code) or down (even)
    lo, hi = BYTES[bits]
    e = torch.frexp(most).exponent.long() - 1 - EMAX[bits]     # of its leading bit, against the last code's
    e = torch.where(past(most * _power(-e)), e + 1, e)
    e = torch.where(most > 0, e, -1000).clamp(lo - 127, hi - 127)
    y = blocks * _power(-e).unsqueeze(-1)
    a = y.abs().clamp(max=float(grid[-1]))
    up = torch.searchsorted(grid, a.contiguous()).clamp(max=grid.numel() - 1)   # first number that is not less
    down = (up - 1).clamp(min=0)
    du, dd = grid[up] - a, a - grid[down]
    code = torch.where(du < dd, up, torch.where(du > dd, down, torch.where(up % 2 == 0, up, down)))
    out = torch.where(y < 0, -grid[code], grid[code]) * _power(e).unsqueeze(-1)
    return out.reshape(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    kind, b, h, n, hd = case["kind"], case["batch"], case["hkv"], case["rows"], case["hd"]
    if kind == "store":
        out = []
        for t in ("k", "v"):
            src = st[t + "_src"]
            got = torch.empty((b, h, n, hd), dtype=torch.float64, device=DEV)
            for i in range(b):
                for j in range(h):
                    got[i, j] = _rounded(src[i, :, j].double(), case[t + "bits"])
            out.append(got)
        return tuple(out)
    if kind == "rows":
        out = []
        for t in ("k", "v"):
            got = torch.empty((b, h, case["ids"], hd), dtype=torch.float64, device=DEV)
            for u in range(b * h):
                i = st["idx"][u].long()
                got[u // h, u % h] = _numbers(st[t][0][u // h, u % h, i], st[t][1][u // h, u % h, i], case[t + "bits"])
            out.append(got)
        return tuple(out)
    heads = h * case["group"]
    out = torch.zeros((b, heads, hd), dtype=torch.float64, device=DEV)
    lse = torch.full((b, heads), -math.inf, dtype=torch.float64, device=DEV)
    new = [torch.zeros((b, h, 1, hd), dtype=torch.float64, device=DEV) for _ in range(2)]
    for i in range(b):
        length = int(st["lens"][i])
        for j in range(h):
            kv = [_numbers(st[t][0][i, j, :length], st[t][1][i, j, :length], case[t + "bits"]) for t in ("k", "v")]
            if kind == "step":
                for which, t in enumerate(("k", "v")):
                    new[which][i, j, 0] = _rounded(st["new_" + t][i, j].double(), case[t + "bits"])
                    kv[which] = torch.cat([kv[which], new[which][i, j]])
            if case["window"]:
                total = kv[0].shape[0]
                keep = list(range(0, min(case["sink"], total)))
                keep += list(range(max(len(keep), total - case["window"]), total))
                kv = [x[torch.tensor(keep, device=DEV)] for x in kv]
            mine = slice(j * case["group"], (j + 1) * case["group"])
            logits = st["q"][i, mine].double() @ kv[0].t() * (1.0 / math.sqrt(hd))
            lse[i, mine] = torch.logsumexp(logits, -1)
            out[i, mine] = torch.softmax(logits, -1) @ kv[1]
    return (out, lse) if kind == "attn" else (out, lse, new[0], new[1])
