"""A paged key/value cache and the attention that reads it: what a program that serves sequences calls once per layer and step.

Two operators, each over a cache in bf16 and over one in 8 bits:
  append     rotates the new rows of q and k by their positions (one axis, or time / height / width) and writes k and v into the pages
             of their sequences; an 8-bit cache has one scale for each page and kv head, which grows with the page
  attention  rows of q against the cached tokens of their sequence, causal, optionally with a sliding window and a few first tokens
             that stay visible: one row per sequence (decode), a few (drafted tokens), or a prompt and its chunks

Sequences have lengths of their own, pages lie in the pool in no order, query heads share kv heads.
"""
import math

import torch

own = False


def listed():
    return [
        # one generated token for each of 16 sequences: the smallest write, latency
        dict(name="append_step", kind="append", cache="bf16", B=16, rows=1, len=1024, H=32, Hkv=8, D=128, page=16, rot=128, pairs="halves", axes=1),
        # prompts of several lengths enter the cache together
        dict(name="append_prompt", kind="append", cache="bf16", B=4, rows=2048, len=2048, H=32, Hkv=8, D=128, page=64, rot=128, pairs="halves", axes=1),
        # one generated token each into an 8-bit cache: the token joins a page that holds tokens already, whose scale may have to grow
        dict(name="append_step_int8", kind="append", cache="int8", B=32, rows=1, len=96, H=32, Hkv=8, D=128, page=32, rot=128, pairs="halves", axes=1),
        # chunks of prompts with images (three axes, a part of each head rotated, neighbouring components paired) into an 8-bit cache
        dict(name="append_chunk_int8_axes", kind="append", cache="int8", B=3, rows=1001, len=1500, H=16, Hkv=4, D=128, page=64, rot=96, pairs="neighbours", axes=3),
        # one token of one sequence over a short context: latency
        dict(name="decode_one", kind="attention", cache="bf16", B=1, rows=1, len=500, H=32, Hkv=8, D=128, page=16, window=0, sinks=0),
        # a batch of sequences of very different lengths, heads in groups of four
        dict(name="decode_batch", kind="attention", cache="bf16", B=16, rows=1, len=8192, H=32, Hkv=8, D=128, page=64, window=0, sinks=0),
        # the same kind of batch over an 8-bit cache
        dict(name="decode_batch_int8", kind="attention", cache="int8", B=24, rows=1, len=8192, H=64, Hkv=8, D=128, page=64, window=0, sinks=0),
        # long contexts of which a window and the first tokens are read
        dict(name="decode_window", kind="attention", cache="bf16", B=32, rows=1, len=16384, H=32, Hkv=8, D=64, page=32, window=2048, sinks=4),
        # drafted tokens of each sequence checked in one call
        dict(name="draft_rows", kind="attention", cache="bf16", B=8, rows=6, len=4096, H=32, Hkv=4, D=128, page=16, window=0, sinks=0),
        # prompts of several lengths on a cache that holds their beginnings: bound by arithmetic
        dict(name="prompt", kind="attention", cache="bf16", B=3, rows=2048, len=4096, H=32, Hkv=8, D=128, page=64, window=0, sinks=0),
        # the same on an 8-bit cache
        dict(name="prompt_int8", kind="attention", cache="int8", B=2, rows=2048, len=3000, H=32, Hkv=8, D=128, page=32, window=0, sinks=0),
        # a long prompt under a window, small heads without sharing
        dict(name="prompt_window", kind="attention", cache="bf16", B=1, rows=6000, len=6000, H=16, Hkv=16, D=64, page=128, window=1000, sinks=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    D = rng.choice([64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8, 8, 16])
    H = Hkv * rng.choice([1, 2, 4, 8] if Hkv > 2 else [4, 7, 8, 16])
    c = dict(kind=rng.choice(["append", "attention", "attention"]), cache=rng.choice(["bf16", "int8"]), H=H, Hkv=Hkv, D=D, page=rng.choice([16, 32, 64, 128]))
    if c["kind"] == "append":
        if rng.random() < 0.5:
            B, rows = _log_int(rng, 1, 64), 1
        else:
            B, rows = _log_int(rng, 1, 6), _log_int(rng, 2, 2048)
            while B * rows * H * D > 4 * 2048 * 32 * 128:
                rows = rows // 2 + 1
        c.update(B=B, rows=rows, len=rows + _log_int(rng, 1, 256))
        c.update(rot=rng.choice([D, D, D // 2, 48]), pairs=rng.choice(["halves", "neighbours"]), axes=rng.choice([1, 1, 3]))
        return c
    how = rng.choice(["one", "one", "few", "prompt", "prompt"])
    if how == "one":
        B = _log_int(rng, 1, 64)
        # at most 0.4 GB of cached values
        c.update(B=B, rows=1, len=min(_log_int(rng, 20, 16384), 100_000_000 // (B * Hkv * D)))
    elif how == "few":
        B = _log_int(rng, 1, 16)
        rows = rng.randint(2, 12)
        c.update(B=B, rows=rows, len=rows + _log_int(rng, 1, 4096))
    else:
        B, rows = _log_int(rng, 1, 4), _log_int(rng, 20, 2048)
        c.update(B=B, rows=rows, len=rows + _log_int(rng, 1, 2000))
        while H * c["B"] * c["rows"] * c["len"] > 32 * 3 * 2048 * 4096:
            c["rows"] = c["rows"] // 2 + 1
            c["len"] = c["len"] // 2 + c["rows"]
    c.update(window=0, sinks=0)
    if rng.random() < 0.4:
        c.update(window=_log_int(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 100]))
    return c


def _spread(most, B, least):
    """B numbers from `most` down to a quarter of it (`least` at the lowest), evenly spread"""
    return [max(least, most - (most - most // 4) * i // max(1, B - 1)) for i in range(B)]


def _plan(c):
    """(rows, tokens in the cache once these rows are in it) of each sequence"""
    rows = _spread(c["rows"], c["B"], 1)
    lens = _spread(c["len"], c["B"], 1)
    return rows, [max(n, r) for n, r in zip(lens, rows)]


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, lens = _plan(c)
    B, H, Hkv, D, P = c["B"], c["H"], c["Hkv"], c["D"], c["page"]
    order = torch.randperm(B, generator=g, device="cuda").tolist()
    rows, lens = [rows[i] for i in order], [lens[i] for i in order]
    need = [-(-n // P) for n in lens]
    pages, width = sum(need) + 3, max(need)
    s = dict(c)
    # pages in no order; entries behind a sequence's last page name no page
    shuffled = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    start = [0]
    for b, n in enumerate(need):
        table[b, :n] = shuffled[sum(need[:b]):sum(need[:b]) + n]
        start.append(start[-1] + rows[b])
    T = start[-1]
    s.update(pages=pages, T=T, max_rows=max(rows), table=table)
    s["row_start"] = torch.tensor(start, dtype=torch.int32, device="cuda") if c["rows"] > 1 else None
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    values = _randn(g, 2, pages, Hkv, P, D, dtype=torch.float32 if c["cache"] == "int8" else torch.bfloat16)
    if c["cache"] == "int8":
        # the tokens that are there have been quantised page by page (all of a page's places hold something)
        s["scale"] = values.abs().amax((3, 4)).div_(127)
        s["kv"] = values.div_(s["scale"][..., None, None]).round_().clamp_(-127, 127).to(torch.int8)
        s["values"] = torch.empty_like(s["kv"], dtype=torch.bfloat16)
    else:
        s["scale"], s["kv"] = None, values
    s["q"] = _randn(g, T, H, D)
    s["out"] = torch.zeros_like(s["q"])
    if c["kind"] == "append":
        # the rows of a fused projection: k and v beside one another.  A token now and then is larger than what its page has seen
        loud = torch.rand(T, 1, 1, generator=g, device="cuda").mul_(2)
        s["k_new"], s["v_new"] = (torch.randn(T, 2 * Hkv, D, generator=g, device="cuda") * loud).to(torch.bfloat16).split(Hkv, 1)
        half, axes, longest = c["rot"] // 2, c["axes"], max(lens)
        turn = torch.arange(longest, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["cos"], s["sin"] = turn.cos().float().contiguous(), turn.sin().float().contiguous()
        # pairs of components for each axis; positions along time, height and width where there are three
        s["section"] = [half] if axes == 1 else [half - 2 * (half // 3), half // 3, half // 3]
        s["positions"] = None if axes == 1 else torch.randint(0, longest, (axes, T), generator=g, device="cuda", dtype=torch.int32)
    return s


def _rows_of(s):
    """sequence and token of each row"""
    row_start = s["row_start"] if s["row_start"] is not None else torch.arange(s["B"] + 1, device="cuda", dtype=torch.int32)
    row = torch.arange(s["T"], device="cuda")
    b = torch.searchsorted(row_start[1:].long(), row, right=True)
    return b, s["seq_lens"].long()[b] - row_start.long()[b + 1] + row


def _rotated(x, s, token):
    """the first `rot` components of each head turned pairwise, in the type of cos and sin"""
    half = s["rot"] // 2
    axis = torch.repeat_interleave(torch.arange(s["axes"], device="cuda"), torch.tensor(s["section"], device="cuda"))
    at = token[:, None].expand(-1, half) if s["positions"] is None else s["positions"].long()[axis].T
    pair = torch.arange(half, device="cuda")
    cos, sin = s["cos"][at, pair][:, None], s["sin"][at, pair][:, None]
    i, j = (pair, pair + half) if s["pairs"] == "halves" else (2 * pair, 2 * pair + 1)
    a, b = x[..., i].to(cos.dtype), x[..., j].to(cos.dtype)
    y = x.to(cos.dtype)
    y[..., i], y[..., j] = a * cos - b * sin, b * cos + a * sin
    return y


def _appended(s, kv, scale):
    """kv ([2, pages, Hkv, page, D]) and scale with the rows in them, and the rotated q, in the type of cos and sin"""
    b, token = _rows_of(s)
    page, place = s["table"].long()[b, token // s["page"]], token % s["page"]
    new = torch.stack([_rotated(s["k_new"], s, token), s["v_new"].to(s["cos"].dtype)])
    q = _rotated(s["q"], s, token)
    if scale is None:
        kv[:, page, :, place] = new.transpose(0, 1).to(kv.dtype)
        return kv, None, q
    largest = torch.zeros_like(scale).index_reduce_(1, page, new.abs().amax(-1), "amax")
    first = torch.full((s["pages"],), s["page"], device="cuda").index_reduce_(0, page, place, "amin")
    before = scale * (first > 0)[:, None]                # a page that begins with a new token has no scale yet
    after = torch.maximum(before, largest / torch.full_like(scale, 127))
    turn = torch.where(after > 0, 1 / after, 0)
    old = torch.arange(s["page"], device="cuda") < first[:, None]
    grown = (after > before)[:, :, :, None, None] & old[None, :, None, :, None] & (first < s["page"])[None, :, None, None, None]
    again = (kv.to(scale.dtype) * before[..., None, None] * turn[..., None, None]).round().clamp(-127, 127)
    kv = torch.where(grown, again, kv.to(scale.dtype))
    kv[:, page, :, place] = (new.transpose(0, 1) * turn[:, page].transpose(0, 1)[..., None]).round().clamp(-127, 127)
    touched = (first < s["page"])[:, None]
    return kv, torch.where(touched, after, scale), q


def _attended(s, dtype):
    """the attention of every row, in the given type; padded to the most rows and the most pages"""
    B, H, Hkv, D, P, R = s["B"], s["H"], s["Hkv"], s["D"], s["page"], s["max_rows"]
    pages = s["table"].long().clamp(min=0)
    kv = s["kv"][:, pages].to(dtype)
    if s["scale"] is not None:
        kv *= s["scale"][:, pages].to(dtype)[..., None, None]
    k, v = kv.transpose(2, 3).reshape(2, B, Hkv, -1, D)
    b, token = _rows_of(s)
    row = token - (s["seq_lens"].long()[b] - torch.bincount(b, minlength=B)[b])
    q = torch.zeros(B, R, H, D, dtype=dtype, device="cuda")
    q[b, row] = s["q"].to(dtype)
    q = q.reshape(B, R, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    score = (q @ k.transpose(-1, -2)).div_(math.sqrt(D)).reshape(B, Hkv, H // Hkv, R, -1)
    place = torch.full((B, R), -1, device="cuda")
    place[b, row] = token
    at = torch.arange(score.shape[-1], device="cuda")
    seen = at <= place[..., None]
    if s["window"]:
        seen &= (at > place[..., None] - s["window"]) | (at < s["sinks"])
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.reshape(B, Hkv, -1, score.shape[-1]) @ v).reshape(B, Hkv, H // Hkv, R, D) / torch.where(total > 0, total, 1)
    return out.permute(0, 3, 1, 2, 4).reshape(B, R, H, D)[b, row]


def _described(s):
    """The library's descriptors of a state's buffers, which a program keeps from step to step."""
    from mm_amx_b200 import capi
    B, H, Hkv, D, P, T = s["B"], s["H"], s["Hkv"], s["D"], s["page"], s["T"]
    es = s["kv"].element_size()
    k, v = s["kv"]
    ks, vs = (None, None) if s["scale"] is None else (t.data_ptr() for t in s["scale"])
    cache = capi.PagedCache(pages=s["pages"], page_tokens=P, Hkv=Hkv, D=D, dtype=capi.BF16 if es == 2 else capi.S8, k=k.data_ptr(), v=v.data_ptr(),
                            page_stride=Hkv * P * D * es, head_stride=P * D * es, token_stride=D * es, k_scale=ks, v_scale=vs, scale_page_stride=Hkv * 4,
                            B=B, max_pages=s["table"].shape[1], page_table=s["table"].data_ptr(), table_stride=s["table"].shape[1] * 4,
                            seq_lens=s["seq_lens"].data_ptr())
    row_start = None if s["row_start"] is None else s["row_start"].data_ptr()
    if s["kind"] == "attention":
        return capi.paged_attention, capi.PagedAttention(
            cache=capi.pointer(cache), T=T, max_rows=s["max_rows"], H=H, row_start=row_start, q=s["q"].data_ptr(), q_row_stride=H * D * 2,
            q_head_stride=D * 2, out=s["out"].data_ptr(), out_row_stride=H * D * 2, out_head_stride=D * 2, scale=1 / math.sqrt(D),
            window=s["window"], sinks=s["sinks"])
    kn, vn = s["k_new"], s["v_new"]
    return capi.kv_append, capi.KvAppend(
        cache=capi.pointer(cache), T=T, row_start=row_start, k=kn.data_ptr(), k_row_stride=kn.stride(0) * 2, k_head_stride=kn.stride(1) * 2,
        v=vn.data_ptr(), v_row_stride=vn.stride(0) * 2, v_head_stride=vn.stride(1) * 2, H=H, q=s["q"].data_ptr(), q_row_stride=H * D * 2,
        q_head_stride=D * 2, q_out=s["out"].data_ptr(), q_out_row_stride=H * D * 2, q_out_head_stride=D * 2, rot_dim=s["rot"],
        interleaved=int(s["pairs"] == "neighbours"), rot_positions=s["cos"].shape[0], rot_cos=s["cos"].data_ptr(), rot_sin=s["sin"].data_ptr(),
        rot_stride=s["cos"].stride(0) * 4, positions=None if s["positions"] is None else s["positions"].data_ptr(), position_stride=T * 4,
        axes=s["axes"], section=(capi.c_int * 3)(*s["section"]))


def _values(s):
    """the cache; in 8 bits as the values it stands for, rounded to bf16 as what reads them does"""
    return s["kv"] if s["scale"] is None else torch.mul(s["kv"], s["scale"][..., None, None], out=s["values"])


def run(state):
    s = state
    if own:
        if "call" not in s:
            s["call"] = _described(s)
        call, what = s["call"]
        call(what)
    elif s["kind"] == "attention":
        s["out"] = _attended(s, torch.float32).to(torch.bfloat16)
    else:
        kv, scale, q = _appended(s, s["kv"], s["scale"])
        s["kv"], s["scale"], s["out"] = kv.to(s["kv"].dtype), scale, q.to(torch.bfloat16)
    return s["out"] if s["kind"] == "attention" else dict(q=s["out"], kv=_values(s))


def exact(case, seed):
    s = prepare(case, seed)
    rows, lens = s["seq_lens"].new_ones(s["B"]) if s["row_start"] is None else s["row_start"].diff(), s["seq_lens"].tolist()
    rows = rows.tolist()
    H, Hkv, D, P = s["H"], s["Hkv"], s["D"], s["page"]
    at = 0
    if s["kind"] == "attention":
        out = torch.zeros(s["T"], H, D, dtype=torch.float64, device="cuda")
        for b in range(s["B"]):
            n, ids = lens[b], s["table"][b, :-(-lens[b] // P)].long()
            for h in range(Hkv):
                k, v = (s["kv"][i, ids, h].double() * (1 if s["scale"] is None else s["scale"][i, ids, h].double()[:, None, None]) for i in (0, 1))
                k, v = k.reshape(-1, D)[:n], v.reshape(-1, D)[:n]
                heads = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
                place = torch.arange(n - rows[b], n, device="cuda")[:, None]
                token = torch.arange(n, device="cuda")[None]
                hidden = token > place
                if s["window"]:
                    hidden |= (token <= place - s["window"]) & (token >= s["sinks"])
                w = torch.einsum("rhd,td->hrt", s["q"][at:at + rows[b], heads].double(), k) * D ** -0.5
                w = torch.softmax(w.masked_fill(hidden, float("-inf")), -1)
                out[at:at + rows[b], heads] = torch.einsum("hrt,td->rhd", w, v)
            at += rows[b]
        return out
    half = s["rot"] // 2
    axis_of = [a for a, n in enumerate(s["section"]) for _ in range(n)]
    cos, sin, column = s["cos"].double(), s["sin"].double(), torch.arange(half, device="cuda")

    def turned(x, token):
        where = torch.stack([token if s["positions"] is None else s["positions"][a].long() for a in axis_of], 1)
        z = torch.complex(cos[where, column], sin[where, column])[:, None]
        x = x.double()
        head, rest = x[..., :s["rot"]], x[..., s["rot"]:]
        if s["pairs"] == "halves":
            y = torch.complex(head[..., :half], head[..., half:]) * z
            return torch.cat([y.real, y.imag, rest], -1)
        y = torch.view_as_complex(head.reshape(*head.shape[:-1], half, 2).contiguous()) * z
        return torch.cat([torch.view_as_real(y).flatten(-2), rest], -1)

    token = torch.cat([torch.arange(n - r, n, device="cuda") for n, r in zip(lens, rows)])
    q, new = turned(s["q"], token), torch.stack([turned(s["k_new"], token), s["v_new"].double()])
    cached = s["kv"].double()
    if s["scale"] is None:
        for b in range(s["B"]):
            t = token[at:at + rows[b]]
            cached[:, s["table"][b, t // P].long(), :, t % P] = new[:, at:at + rows[b]].transpose(0, 1)
            at += rows[b]
        return dict(q=q, kv=cached)
    scale = s["scale"].double()
    for b in range(s["B"]):
        first = lens[b] - rows[b]
        for i in range(first // P, -(-lens[b] // P)):
            lo, hi = max(first, i * P), min(lens[b], (i + 1) * P)
            page, part = int(s["table"][b, i]), new[:, at + lo - first:at + hi - first].transpose(1, 2)
            largest = part.abs().amax((2, 3)) / 127
            before = scale[:, page] if lo > i * P else torch.zeros_like(largest)
            after = torch.maximum(before, largest)
            if lo > i * P:
                again = (cached[:, page, :, :lo - i * P] * (before / after)[..., None, None]).round()
                cached[:, page, :, :lo - i * P] = torch.where((after > before)[..., None, None], again, cached[:, page, :, :lo - i * P])
            cached[:, page, :, lo - i * P:hi - i * P] = (part / after[..., None, None].clamp(min=1e-300)).round()
            scale[:, page] = after
        at += rows[b]
    return dict(q=q, kv=cached * scale[..., None, None])


def work(case):
    c = case
    rows, lens = _plan(c)
    H, Hkv, D, P = c["H"], c["Hkv"], c["D"], c["page"]
    es, T = (1 if c["cache"] == "int8" else 2), sum(rows)
    table = 4 * sum(-(-n // P) for n in lens) + 8 * c["B"]
    if c["kind"] == "append":
        touched = sum(-(-n // P) - (n - r) // P for n, r in zip(lens, rows))
        scales = touched * Hkv * 2 * 8 if c["cache"] == "int8" else 0
        turns = T * c["rot"] * 4
        return dict(bytes=T * H * D * 4 + T * Hkv * D * 2 * (2 + es) + scales + turns + 4 * touched, flops=T * (H + Hkv) * c["rot"] * 3)
    window, sinks = c["window"], c["sinks"]
    seen = read = 0
    for r, n in zip(rows, lens):
        if not window:
            seen += r * n - r * (r - 1) // 2
            read += n
        else:
            seen += sum(min(p + 1, window) + max(0, min(sinks, p + 1 - window)) for p in range(n - r, n))
            low = max(0, n - r - window + 1)
            read += n - low + min(sinks, low)
    scales = -(-read // P) * Hkv * 8 if c["cache"] == "int8" else 0
    return dict(bytes=2 * read * Hkv * D * es + scales + 2 * T * H * D * 2 + table, flops=4 * seen * H * D)
