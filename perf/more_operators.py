"""The paged cache: what is measured of it, over which ranges, and its operators in their plain form.

K and V of a layer lie in pages of ``page`` rows, (n_pages, hkv, page, hd) bf16; ``table`` (batch, pages of the longest
sequence) int32 names the page of every ``page`` rows of a sequence, -1 where it has none.  ``start`` (batch) int32: the
rows that a sequence held before its new tokens; token i of sequence b is its row start[b] + i.  New tokens come packed
(tokens of all sequences one after another, those of sequence b from cu[b] to cu[b + 1]) or one to a sequence.  The kinds:

  append  K and V of new tokens written into their pages, K and the queries rotated by their positions on the way
  decode  one new token's attention over the rows of its sequence, its own among them
  chunk   the same for several new tokens of a sequence, each over the rows up to its own

A case is a dict of plain values: kind, batch, hkv, group, hd, page, rows (the longest sequence, new tokens included), new (the
most new tokens of a sequence), ragged (sequences of other lengths and other numbers of tokens), sink, window (rows
attended: the first ``sink`` and the last ``window`` up to the token; 0: all of them), and of an append rot (rotated
columns), axes (positions of a token: 1, its row, or 3, time, height and width), interleaved (pairs of adjacent columns).
"""
import math

import torch

own = False

DEV = "cuda"
THETA = 500000.0


def _case(name, kind, batch, hkv, group, hd, page, rows, new, ragged=False, sink=0, window=0, rot=0, axes=1, interleaved=False):
    return dict(name=name, kind=kind, batch=batch, hkv=hkv, group=group, hd=hd, page=page, rows=rows, new=new, ragged=ragged,
                sink=sink, window=window, rot=rot, axes=axes, interleaved=interleaved)


def listed():
    return [
        # a decode step's tokens of a served batch: latency
        _case("append_step_8x4k", "append", 8, 8, 4, 128, 16, 4096, 1, ragged=True, rot=128),
        # a document of about 32K tokens
        _case("append_doc_32k", "append", 1, 8, 4, 128, 64, 32601, 32601, rot=128),
        # prompts of text and images, positions in time, height and width
        _case("append_images_5x4k", "append", 5, 8, 4, 128, 32, 4099, 4099, ragged=True, rot=128, axes=3),
        # a token of a chat turn: latency
        _case("attn_chat_517", "decode", 1, 8, 4, 128, 16, 517, 1),
        # one document of about 32K tokens
        _case("attn_doc_32k", "decode", 1, 8, 4, 128, 64, 32601, 1),
        # narrow heads in groups of seven, sequences of many lengths
        _case("attn_ragged_5x16k", "decode", 5, 4, 7, 64, 32, 16391, 1, ragged=True),
        # batched serving at 128K tokens
        _case("attn_serve_8x128k", "decode", 8, 8, 4, 128, 64, 131072, 1),
        # a chat turn's prompt: latency
        _case("chunk_chat_517", "chunk", 1, 8, 4, 128, 16, 517, 517),
        # a prompt of 8K tokens
        _case("chunk_prompt_8k", "chunk", 1, 8, 4, 128, 64, 8195, 8195),
        # the next 2K tokens of a document that holds about 30K
        _case("chunk_doc_2k_of_32k", "chunk", 1, 8, 4, 128, 64, 32601, 2048),
        # a served batch of prompts behind shared or cached prefixes, a decoding sequence among them
        _case("chunk_ragged_5x16k", "chunk", 5, 4, 7, 64, 32, 16391, 1021, ragged=True),
        # four drafted tokens of every sequence of a batch
        _case("chunk_draft_8x4_of_32k", "chunk", 8, 8, 4, 128, 64, 32601, 4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "chunk", "chunk", "chunk"])
    most = [max(_cost(c)[i] for c in listed() if c["kind"] == kind) for i in range(3)]
    while True:
        hd = rng.choice([64, 128, 128, 256])
        c = _case("", kind, _log_int(rng, 1, 16), rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16]), hd,
                  rng.choice([16, 32, 64, 128, 256]), _log_int(rng, 2, 32768 if kind == "append" else 131072), 1)
        del c["name"]
        c["ragged"] = rng.random() < 0.5
        if kind == "chunk" or (kind == "append" and rng.random() < 0.6):
            c["new"] = _log_int(rng, 2, min(c["rows"], 32768 if kind == "append" else 8192))
        if kind == "append":
            c["rot"] = rng.choice([hd, hd, hd // 2, hd // 4])
            c["axes"], c["interleaved"] = rng.choice([1, 3]), rng.random() < 0.3
        elif rng.random() < 0.3:
            c["sink"], c["window"] = rng.choice([0, 1, 4, 64]), _log_int(rng, 1, c["rows"] + 1)
        if all(x <= y for x, y in zip(_cost(c), most)):
            return c


# ---- the cases ------------------------------------------------------------------------------------------------------

def _lengths(case):
    """(rows held before, new tokens) of every sequence; whole numbers of the case alone."""
    n, new, b = case["rows"], case["new"], case["batch"]
    if not case["ragged"]:
        return [n - new] * b, [new] * b
    share = [((i + 1) * 0.6180339887498949) % 1.0 for i in range(b)]
    counts = [max(1, int(new * s)) for s in share]
    starts = [int((n - c) * ((s * 7.389) % 1.0)) for c, s in zip(counts, share)]
    if b > 1 and case["kind"] == "chunk":
        counts[0] = 1                       # a decoding sequence
    counts[b // 2], starts[b // 2] = new, n - new
    return starts, counts


def _sections(case):
    """Frequencies that go by time, height and width."""
    half = case["rot"] // 2
    return (half - 2 * (3 * half // 8), 3 * half // 8, 3 * half // 8)


def _cost(case):
    """Bytes, operations, and numbers that the plain form holds at once."""
    w = work(case)
    held = case["batch"] * case["hkv"] * case["rows"] * case["hd"]
    return w["bytes"], w["flops"], held + case["batch"] * case["hkv"] * case["group"] * case["rows"] * case["new"] * (case["kind"] != "append")


def _numbers(shape, g):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    b, h, group, hd, page, n = (case[x] for x in ("batch", "hkv", "group", "hd", "page", "rows"))
    hq, kind = h * group, case["kind"]
    starts, counts = _lengths(case)
    wide = (n + page - 1) // page
    st = {"case": case, "scale": 1.0 / math.sqrt(hd), "tokens": sum(counts)}
    # every sequence's pages, in any order; -1 behind its last row; some pages are no one's
    have = [(s + c + page - 1) // page for s, c in zip(starts, counts)]
    n_pages = sum(have) + 3
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((b, wide), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, p in enumerate(have):
        table[i, :p] = order[at:at + p]
        at += p
    st["table"] = table
    st["start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    st["cu"] = torch.tensor(ends, dtype=torch.int32, device=DEV)
    if kind == "append":
        # what a model's projection leaves: queries, keys and values of a token one behind the other
        st["qkv"] = _numbers((sum(counts), (hq + 2 * h) * hd), g)
        st["k"] = torch.zeros((n_pages, h, page, hd), dtype=torch.bfloat16, device=DEV)
        st["v"] = torch.zeros_like(st["k"])
        half = case["rot"] // 2
        st["inv_freq"] = 1.0 / (THETA ** (torch.arange(half, device=DEV, dtype=torch.float32) / half))
        if case["axes"] == 3:
            # rows of patches, as many to a row as the seed says, behind some text
            row = torch.cat([torch.arange(s, s + c, device=DEV) for s, c in zip(starts, counts)])
            width = int(torch.randint(16, 65, (1,), generator=g, device=DEV))
            text = row < 64
            pos = torch.stack([torch.where(text, row, 64), torch.where(text, row, 64 + (row - 64) // width),
                               torch.where(text, row, 64 + (row - 64) % width)], -1)
            st["pos"] = pos.to(torch.int32)
    else:
        st["k"] = _numbers((n_pages, h, page, hd), g)
        # keys with channels of unequal size (log-normal), as keys have them
        st["k"].mul_(torch.exp(torch.randn((hd,), generator=g, device=DEV)).to(torch.bfloat16))
        st["v"] = _numbers((n_pages, h, page, hd), g)
        st["q"] = _numbers((sum(counts), hq, hd), g)
    return st


def _sequence_of(st):
    """The sequence of every packed token, its number there, and its row."""
    at = torch.arange(st["tokens"], device=DEV)
    seq = torch.searchsorted(st["cu"], at.to(torch.int32), right=True) - 1
    i = at - st["cu"].long()[seq]
    return seq, i, st["start"].long()[seq] + i


def _rotate(x, cos, sin, rot, interleaved):
    """x (tokens, heads, hd) in fp32; cos, sin (tokens, rot / 2)."""
    cos, sin = cos.unsqueeze(1), sin.unsqueeze(1)
    y, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y.chunk(2, -1)
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, rest], -1)


def _dense(pages, table):
    """The rows of every sequence, (batch, hkv, rows, hd) fp32; those without a page are of any page."""
    x = pages[table.long().clamp(min=0)]                    # (batch, pages, hkv, page, hd)
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3).float()


def run(state):
    case, st = state["case"], state
    b, h, group, hd, page, new = (case[x] for x in ("batch", "hkv", "group", "hd", "page", "new"))
    hq = h * group
    cu = None if new == 1 else st["cu"]                     # without it: one token of every sequence
    if case["kind"] == "append":
        q, k, v = (x.unflatten(-1, (-1, hd)) for x in st["qkv"].split([hq * hd, h * hd, h * hd], -1))
    if own:
        from diffcache_amd import _hip as hip
        if case["kind"] == "append":
            out = hip.paged_append(st["k"], st["v"], st["table"], k, v, st["start"], cu=cu, max_new=new, q=q,
                                   inv_freq=st["inv_freq"], interleaved=case["interleaved"], pos=st.get("pos"),
                                   sections=_sections(case) if case["axes"] == 3 else None)
            return st["k"], st["v"], out
        return hip.paged_attn(st["q"], st["k"], st["v"], st["table"], st["start"], cu=cu, max_new=new, n_rows=case["rows"],
                              n_sink=case["sink"], window=case["window"], want_lse=True)
    seq, i, row = _sequence_of(st)
    if case["kind"] == "append":
        pos = st["pos"] if case["axes"] == 3 else row.unsqueeze(-1)
        which = torch.arange(case["rot"] // 2, device=DEV)
        if case["axes"] == 3:
            t, hh, _ = _sections(case)
            which = (which >= t).long() + (which >= t + hh).long()
        else:
            which = which * 0
        angle = pos[:, which].double() * st["inv_freq"].double()
        cos, sin = angle.cos().float(), angle.sin().float()
        at = st["table"].long()[seq, row // page]
        st["k"][at, :, row % page] = _rotate(k.float(), cos, sin, case["rot"], case["interleaved"]).to(torch.bfloat16)
        st["v"][at, :, row % page] = v
        return st["k"], st["v"], _rotate(q.float(), cos, sin, case["rot"], case["interleaved"]).to(torch.bfloat16)
    # the queries of every sequence, padded to as many tokens: (batch, hkv, new * group, hd)
    at = (st["cu"].long()[:-1, None] + torch.arange(new, device=DEV)).clamp(max=st["tokens"] - 1)
    q = st["q"].float()[at].view(b, new, h, group, hd).transpose(1, 2).reshape(b, h, new * group, hd)
    k, v = _dense(st["k"], st["table"]), _dense(st["v"], st["table"])
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(st["scale"]).view(b, h, new, group, -1)
    own_row = (st["start"].long()[:, None] + torch.arange(new, device=DEV)).unsqueeze(-1)   # (batch, new, 1)
    rows = torch.arange(k.shape[2], device=DEV)
    live = rows <= own_row
    if case["window"]:
        live &= (rows < case["sink"]) | (rows > own_row - case["window"])
    s.masked_fill_(~live.view(b, 1, new, 1, -1), -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, h, new * group, -1), v).view(b, h, new, group, hd) / total
    lse = (m + total.log()).squeeze(-1)                     # (batch, hkv, new, group)
    return (out.permute(0, 2, 1, 3, 4)[seq, i].reshape(-1, hq, hd).to(torch.bfloat16),
            lse.permute(0, 2, 1, 3)[seq, i].reshape(-1, hq))


def _attended(case):
    """Rows that all tokens attend to, of one head, and rows that a head has to read."""
    total = read = 0
    sink, window = case["sink"], case["window"]
    for s, c in zip(*_lengths(case)):
        if window:
            total += sum(min(x, sink + window) for x in range(s + 1, s + c + 1))
            first = max(0, s + 1 - window)                  # of the first token's window
            read += min(sink, first) + s + c - first
        else:
            total += c * s + c * (c + 1) // 2
            read += s + c
    return total, read


def work(case):
    b, h, group, hd = (case[x] for x in ("batch", "hkv", "group", "hd"))
    tokens = sum(_lengths(case)[1])
    if case["kind"] == "append":    # queries, keys and values in and out; three operations to a rotated number
        return {"bytes": tokens * (4 * (group + 2) * h * hd + 4 * case["axes"]), "flops": tokens * (group + 1) * h * case["rot"] * 3}
    total, read = _attended(case)
    return {"bytes": h * read * 4 * hd + tokens * h * group * (4 * hd + 4) + 4 * b * ((case["rows"] - 1) // case["page"] + 1),
            "flops": h * group * total * 4 * hd}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _pages_of(st, i, n):
    """Page and row there of rows 0 .. n - 1 of sequence i."""
    r = torch.arange(n, device=DEV)
    page = st["case"]["page"]
    return st["table"][i].long()[r // page], r % page


def exact(case, seed):
    st = prepare(case, seed)
    h, group, hd = case["hkv"], case["group"], case["hd"]
    starts, counts = _lengths(case)
    ends = st["cu"].tolist()
    if case["kind"] == "append":
        half = case["rot"] // 2
        heads = st["qkv"].double().unflatten(-1, (-1, hd))
        freq = st["inv_freq"].double()
        turned = heads.clone()
        lo = 0
        spans = _sections(case) if case["axes"] == 3 else (half,)
        for axis, span in enumerate(spans):
            for j in range(lo, lo + span):
                if case["axes"] == 3:
                    pos = st["pos"][:, axis].double()
                else:
                    pos = torch.cat([torch.arange(s, s + c, device=DEV) for s, c in zip(starts, counts)]).double()
                a, b = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + half)
                z = torch.complex(heads[..., a], heads[..., b]) * torch.polar(torch.ones_like(pos), pos * freq[j])[:, None]
                turned[..., a], turned[..., b] = z.real, z.imag
            lo += span
        k, v = st["k"].double(), st["v"].double()
        for i, (s, c) in enumerate(zip(starts, counts)):
            at, slot = (x[s:] for x in _pages_of(st, i, s + c))
            k[at, :, slot] = turned[ends[i]:ends[i + 1], h * group:h * group + h]
            v[at, :, slot] = heads[ends[i]:ends[i + 1], h * group + h:]
        return k, v, turned[:, :h * group].contiguous()
    out = torch.zeros((st["tokens"], h * group, hd), dtype=torch.float64, device=DEV)
    lse = torch.zeros((st["tokens"], h * group), dtype=torch.float64, device=DEV)
    for i, (s, c) in enumerate(zip(starts, counts)):
        at, slot = _pages_of(st, i, s + c)
        for j in range(h):
            k, v = st["k"][at, j, slot].double(), st["v"][at, j, slot].double()
            for lo in range(0, c, 1024):
                hi = min(lo + 1024, c)
                upto = s + hi
                mine = st["q"][ends[i] + lo:ends[i] + hi, j * group:(j + 1) * group].double().flatten(0, 1)
                logits = (mine @ k[:upto].t() / math.sqrt(hd)).view(hi - lo, group, upto)
                last = torch.arange(s + lo, upto, device=DEV)[:, None, None]
                r = torch.arange(upto, device=DEV)
                hidden = r > last
                if case["window"]:
                    hidden |= (r <= last - case["window"]) & (r >= case["sink"])
                logits = logits.masked_fill(hidden, -math.inf)
                at_ = slice(ends[i] + lo, ends[i] + hi)
                lse[at_, j * group:(j + 1) * group] = torch.logsumexp(logits, -1)
                out[at_, j * group:(j + 1) * group] = (torch.softmax(logits, -1).flatten(0, 1) @ v[:upto]).view(hi - lo, group, hd)
    return out, lse
