"""Cases of the attention operators next to the MoE layers: rotary positions, the append into the paged 8-bit
key/value cache, and attention over that cache. `run` computes them in elementary torch operations, or, where `own`
is true, through eva_b200.attention.

Cache: pages of 64 tokens; keys e4m3 [pages, heads, 64, key_dim], values e4m3 [pages, heads, value_dim, 64], one
power-of-two scale (e8m0) per block of 16 tokens and head. A batch is ragged: sequence b has the token rows
q_start[b] .. q_start[b + 1] - 1, which are the last ones of its seq_lens[b] tokens.
"""
import math

import torch

own = False

PAGE, BLOCK = 64, 16
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases --------------------------------------------------------------------------------------------------

def _rotate(name, tokens, heads, dim, rot, offset, layout, dtype, scaling="none", inverse=False, far=4096):
    return dict(name=name, op="rotate", tokens=tokens, heads=heads, dim=dim, rot=rot, offset=offset, layout=layout,
                dtype=dtype, scaling=scaling, inverse=inverse, far=far)


def _append(name, seqs, new, context, kv_heads, key_dim, value_dim, layout, dtype, ragged):
    return dict(name=name, op="append", seqs=seqs, new=new, context=context, kv_heads=kv_heads, key_dim=key_dim,
                value_dim=value_dim, layout=layout, dtype=dtype, ragged=ragged)


def _attend(name, seqs, new, context, heads, kv_heads, key_dim, value_dim, dtype, ragged, window=0):
    return dict(name=name, op="attend", seqs=seqs, new=new, context=context, heads=heads, kv_heads=kv_heads,
                key_dim=key_dim, value_dim=value_dim, dtype=dtype, ragged=ragged, window=window)


def listed():
    return [
        # the query of one decoding token: pure latency
        _rotate("rotate token", 1, 16, 128, 128, 0, "half", "bf16"),
        # a prompt's queries, rotated in the last 64 of 192 dimensions, scaled for long contexts
        _rotate("rotate prompt", 8192, 32, 192, 64, 128, "interleaved", "bf16", "yarn", False, 160000),
        # the gradient's rotation in 32 bits: odd token and head counts, a rotated part in the middle
        _rotate("rotate back", 3001, 5, 80, 40, 8, "half", "fp32", "linear", True, 1000000),
        # a decode step of 32 sequences: one token each, into blocks that are partly full
        _append("append step", 32, 1, 4000, 8, 128, 128, "half", "bf16", True),
        # ragged prompts, some behind a context that ends inside a block
        _append("append prompts", 7, 4096, 300, 16, 192, 128, "interleaved", "fp16", True),
        # one short conversation, one token: pure latency
        _attend("attend token", 1, 1, 150, 8, 2, 64, 64, "bf16", False),
        # a decode step of 64 sequences of very different lengths
        _attend("attend step", 64, 1, 8192, 32, 8, 128, 128, "bf16", True),
        # two long documents
        _attend("attend long", 2, 1, 131071, 64, 8, 128, 128, "bf16", False),
        # four drafted tokens to check for each sequence, within a window
        _attend("attend draft", 16, 4, 6000, 16, 4, 128, 128, "fp16", True, 4096),
        # a prompt from its first token on
        _attend("attend prompt", 1, 8192, 0, 16, 4, 128, 128, "bf16", False),
        # pieces of prompts behind long contexts, a key and a value head for each query head
        _attend("attend pieces", 3, 700, 20000, 16, 16, 192, 128, "bf16", True),
        # rotate the query, append, attend: a whole decode step of one layer
        dict(_attend("step", 24, 1, 3000, 32, 8, 128, 128, "bf16", True), op="step", layout="half"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotate", "append", "attend", "attend", "attend", "step"))
    layout = rng.choice(("half", "interleaved"))
    if op == "rotate":
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        rot = 2 * rng.randint(8, 64)
        offset = 2 * rng.randint(0, 32)
        dim = rot + offset + 2 * rng.randint(0, 16)
        return _rotate("", _log(rng, 1, 6000), rng.randint(1, 32), dim, rot, offset, layout, dtype,
                       rng.choice(("none", "linear", "yarn")), rng.random() < 0.3, _log(rng, 100, 2000000))
    key_dim, value_dim = rng.choice(((64, 64), (128, 128), (192, 128)))
    dtype = rng.choice(("bf16", "fp16"))
    kv_heads = rng.randint(1, 12)
    if op == "append":
        seqs = _log(rng, 1, 48)
        new = _log(rng, 1, 8000 // seqs)
        return _append("", seqs, new, _log(rng, 1, 4000) - 1, kv_heads, key_dim, value_dim, layout, dtype,
                       rng.random() < 0.7)
    group = rng.choice((1, 2, 3, 4, 5, 8))
    window = rng.choice((0, 0, _log(rng, 1, 5000)))
    seqs = _log(rng, 1, 64)
    if op == "step":
        return dict(_attend("", seqs, 1, _log(rng, 1, 120000 // seqs), kv_heads * group, kv_heads, key_dim, value_dim,
                            dtype, rng.random() < 0.7, window), op="step", layout=layout)
    new = rng.choice((1, 1, rng.randint(1, 8), _log(rng, 8, 2000)))
    if new > 8:
        seqs = min(seqs, 4)
    return _attend("", seqs, new, _log(rng, 1, max(2, 100000 // (seqs * (1 + new // 200)))) - 1, kv_heads * group,
                   kv_heads, key_dim, value_dim, dtype, rng.random() < 0.7, window)


# ---- inputs -------------------------------------------------------------------------------------------------

def _inv_freq(rot, scaling):
    """Angle per position of each pair, in Python floats, and the factor on cos and sin."""
    base, factor, original = 10000.0, 40.0, 4096
    f = [base ** (-2 * i / rot) for i in range(rot // 2)]
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return [x / 8.0 for x in f], 1.0
    at = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
    keep = [1.0 - min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in range(rot // 2)]
    return [x / factor * (1.0 - s) + x * s for x, s in zip(f, keep)], 0.1 * math.log(factor) + 1.0


def _lengths(case):
    """New tokens and total lengths of the sequences: the last one has the case's, a ragged batch's others spread below."""
    n, c, seqs = case["new"], case["context"], case["seqs"]
    if not case["ragged"]:
        return [n] * seqs, [n + c] * seqs
    at = [(b * 0.6180339887 + 0.31) % 1.0 for b in range(seqs)]
    new = [max(1, round(n * (0.1 + 0.9 * x))) for x in at[:-1]] + [n]
    ctx = [round(c * ((7 * x + 0.17) % 1.0)) for x in at[:-1]] + [c]
    return new, [a + b for a, b in zip(new, ctx)]


def _quantise(x, tokens_dim):
    """Values of a cache in blocks of 16 along tokens_dim: e4m3 codes and the power-of-two scales' exponents."""
    y = x.unflatten(tokens_dim, (PAGE // BLOCK, BLOCK))
    amax = y.abs().amax(dim=(y.dim() - 1, tokens_dim + 1) if tokens_dim == 2 else (2, y.dim() - 1))
    e = _exponent(amax)
    shape = [1] * y.dim()
    shape[0], shape[1], shape[tokens_dim] = y.shape[0], y.shape[1], y.shape[tokens_dim]
    return (y * torch.exp2(-e.float()).view(shape)).to(E4M3).flatten(tokens_dim, tokens_dim + 1), e


def _exponent(amax):
    """Smallest e with amax <= 448 * 2^e, from the bits of amax (32-bit floats), between -126 and 127."""
    bits = amax.float().view(torch.int32)
    e = (bits >> 23) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000).int()
    return e.clamp(-126, 127)


def _scale_codes(e):
    return (e + 127).to(torch.uint8).view(E8M0)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    dt = DTYPES[case["dtype"]]
    s = {"op": case["op"], "dtype": dt}
    if case["op"] == "rotate":
        s["x"] = rand(case["tokens"], case["heads"], case["dim"]).to(dt)
        s["positions"] = torch.randint(0, case["far"], (case["tokens"],), generator=g, device=dev)
        freq, mscale = _inv_freq(case["rot"], case["scaling"])
        s.update(layout=case["layout"], offset=case["offset"], rot=case["rot"], inverse=case["inverse"], mscale=mscale)
        scaling = case["scaling"]
    else:
        heads, dk, dv = case["kv_heads"], case["key_dim"], case["value_dim"]
        new, lens = _lengths(case)
        each = [-(-n // PAGE) for n in lens]
        pages = sum(each) + 3
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((len(lens), max(each)), -1, dtype=torch.int32)   # no page behind a sequence's last one
        for b, n in enumerate(each):
            table[b, :n] = torch.tensor(order[:n], dtype=torch.int32)
            order = order[n:]
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        T = start[-1]
        # keys with a few loud channels, as trained heads have; every page is full of some earlier use's tokens
        loud = 1 + 6 * (torch.rand(heads, 1, dk, generator=g, device=dev) > 0.95)
        s["k"], ke = _quantise(rand(pages, heads, PAGE, dk) * loud, 2)
        s["v"], ve = _quantise(rand(pages, heads, dv, PAGE) * 0.5, 3)
        s["ks"], s["vs"] = _scale_codes(ke), _scale_codes(ve)
        s["q_start"] = torch.tensor(start, dtype=torch.int32, device=dev)
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["table"] = table.to(dev)
        s["max_q"] = max(new)
        s["window"] = case.get("window", 0)
        s["scale"] = dk ** -0.5
        if case["op"] != "append":
            s["q"] = (rand(T, case["heads"], dk) * (1 + 2 * torch.rand(1, case["heads"], 1, generator=g, device=dev))).to(dt)
        if case["op"] != "attend":
            # slices of one projection's rows, as a model has them
            kv = torch.cat([(rand(T, heads, dk) * loud.view(1, heads, dk)).flatten(1), rand(T, heads * dv) * 0.5], 1).to(dt)
            s["new_k"] = kv[:, :heads * dk].unflatten(1, (heads, dk))
            s["new_v"] = kv[:, heads * dk:].unflatten(1, (heads, dv))
            rot = dk if case["layout"] == "half" else dk - dk // 3 * 2   # the whole key, or its last part
            rot -= rot % 2
            freq, mscale = _inv_freq(rot, "none")
            s.update(layout=case["layout"], offset=dk - rot, rot=rot, inverse=False, mscale=mscale)
            scaling = "none"
            s["positions"] = torch.cat([torch.arange(n - m, n) for m, n in zip(new, lens)]).to(dev)
    if case["op"] != "attend":
        s["freq"] = torch.tensor(freq, dtype=torch.float64, device=dev)
    if own:
        from eva_b200.attention import PagedBatch, PagedKVCache, Rotary
        if case["op"] != "attend":
            more = {"none": {}, "linear": {"factor": 8.0}, "yarn": {"factor": 40.0, "original_len": 4096}}[scaling]
            s["rotary"] = Rotary(s["rot"], base=10000.0, layout=s["layout"], offset=s["offset"], scaling=scaling,
                                 device=dev, **more)
        if case["op"] != "rotate":
            s["cache"] = PagedKVCache(pages, heads, dk, dv, device=dev, k=s["k"], v=s["v"], k_scale=s["ks"],
                                      v_scale=s["vs"])
            s["batch"] = PagedBatch(s["q_start"], s["seq_lens"], s["table"], s["max_q"])
    return s


# ---- the operators ------------------------------------------------------------------------------------------

def _rotated(x, positions, freq, mscale, layout, offset, rot, inverse):
    """x [tokens, heads, dim] in 32 bits, rotated; the angles in 64 bits."""
    a = positions.double()[:, None] * freq
    c = (a.cos() * mscale).float()[:, None, :]
    n = (a.sin() * (-mscale if inverse else mscale)).float()[:, None, :]
    x = x.float()
    part = x[..., offset:offset + rot]
    if layout == "half":
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        part = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    return torch.cat([x[..., :offset], part, x[..., offset + rot:]], -1)


def _rows_of(s, tokens):
    """Sequence and place within its new tokens of each token row."""
    t = torch.arange(tokens, device=s["q_start"].device)
    b = torch.searchsorted(s["q_start"].long(), t, right=True) - 1
    return b, t - s["q_start"].long()[b]


def _append_plain(s):
    """Requantises every block of 16 tokens that gets a token: the old ones in it and the new ones."""
    dev, new_k, new_v = s["k"].device, s["new_k"], s["new_v"]
    T, B = new_k.shape[0], s["seq_lens"].numel()
    key = _rotated(new_k, s["positions"], s["freq"], s["mscale"], s["layout"], s["offset"], s["rot"], False)
    val = new_v.float()
    key = torch.where(key.isfinite().all(-1, keepdim=True) & val.isfinite().all(-1, keepdim=True), key, math.nan)
    val = torch.where(val.isfinite(), val, 0.0)
    start, lens = s["q_start"].long(), s["seq_lens"].long()
    ctx = lens - (start[1:] - start[:-1])
    n_blocks = (s["max_q"] + BLOCK - 2) // BLOCK + 1
    block = ctx[:, None] // BLOCK + torch.arange(n_blocks, device=dev)             # [B, n]
    pos = block[..., None] * BLOCK + torch.arange(BLOCK, device=dev)               # [B, n, 16]
    is_new = (pos >= ctx[:, None, None]) & (pos < lens[:, None, None])
    is_old = (pos < ctx[:, None, None]) & is_new.any(-1, keepdim=True)
    src = (start[:-1, None, None] + pos - ctx[:, None, None]).clamp(0, T - 1)
    page = s["table"].long().gather(1, (block // 4).clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    at = block % 4
    touched = is_new.any(-1)                                                       # [B, n]
    keep = is_new | is_old
    slot = torch.arange(BLOCK, device=dev)
    # keys: [B, n, H, 16, D], values the same
    page_i, tok_i = page[..., None], at[..., None] * BLOCK + slot
    for codes, scales, rows, is_key in ((s["k"], s["ks"], key, True), (s["v"], s["vs"], val, False)):
        raw = codes[page_i, :, tok_i] if is_key else codes[page_i, :, :, tok_i]    # [B, n, 16, H, D]
        e_old = scales.view(torch.uint8)[page, :, at].int() - 127                  # [B, n, H]
        old = raw.float()
        fresh = rows[src]                                                          # [B, n, 16, H, D]
        finite = torch.where(is_new[..., None, None] & fresh.isfinite(), fresh.abs(), 0.0)
        e = _exponent(finite.amax(dim=(2, 4)))
        e = torch.where(is_old.any(-1)[..., None], torch.maximum(e, e_old), e)
        down = torch.exp2((e_old - e).float())[:, :, None, :, None]
        put = torch.where(is_new[..., None, None], fresh * torch.exp2(-e.float())[:, :, None, :, None],
                          torch.where(is_old[..., None, None], old * down, 0.0)).to(E4M3).view(torch.uint8)
        put = torch.where(keep[..., None, None], put, raw.view(torch.uint8))
        sel = touched.nonzero(as_tuple=True)
        bytes_ = codes.view(torch.uint8)
        if is_key:
            bytes_[page_i[sel], :, tok_i[sel]] = put[sel]
        else:
            bytes_[page_i[sel], :, :, tok_i[sel]] = put[sel]
        scales.view(torch.uint8)[page[sel], :, at[sel]] = (e[sel] + 127).to(torch.uint8)


def _attend_plain(s, q):
    k, v, table, lens = s["k"], s["v"], s["table"].long().clamp(min=0), s["seq_lens"].long()
    T, heads, dk = q.shape
    kv_heads, dv, B, L = k.shape[1], v.shape[2], table.shape[0], table.shape[1] * PAGE
    g, mq, start = heads // kv_heads, s["max_q"], s["q_start"].long()
    n = start[1:] - start[:-1]
    i = torch.arange(mq, device=q.device)
    rows = (start[:-1, None] + i).clamp(max=T - 1)
    qp = q[rows].float().unflatten(2, (kv_heads, g)).permute(0, 2, 1, 3, 4).reshape(B, kv_heads, mq * g, dk)
    keys = k[table].float() * s["ks"][table].float().repeat_interleave(BLOCK, -1)[..., None]
    keys = keys.permute(0, 2, 1, 3, 4).reshape(B, kv_heads, L, dk)
    vals = v[table].float() * s["vs"][table].float().repeat_interleave(BLOCK, -1)[..., None, :]
    vals = vals.permute(0, 2, 1, 4, 3).reshape(B, kv_heads, L, dv)
    j = torch.arange(L, device=q.device)
    vals = torch.where((j < lens[:, None])[:, None, :, None], vals, 0.0)
    pos = lens[:, None] - n[:, None] + i                                           # [B, mq]
    seen = j <= pos[..., None]
    if s["window"]:
        seen &= j > pos[..., None] - s["window"]
    seen = seen.repeat_interleave(g, 1)[:, None]                                   # [B, 1, mq g, L]
    x = torch.matmul(qp, keys.transpose(2, 3)) * s["scale"]
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, vals) / torch.where(total == 0, 1.0, total)
    o = o.view(B, kv_heads, mq, g, dv).permute(0, 2, 1, 3, 4).reshape(B, mq, heads, dv)
    b, at = _rows_of(s, T)
    return o[b, at].to(s["dtype"])


def run(s):
    if own:
        if s["op"] == "rotate":
            return s["rotary"].apply(s["x"], s["positions"], inverse=s["inverse"])
        q = s.get("q")
        if s["op"] != "attend":
            if s["op"] == "step":
                q = s["rotary"].apply(q, s["positions"])
            s["cache"].append(s["new_k"], s["new_v"], s["batch"], rotary=s["rotary"])
            if s["op"] == "append":
                return s["k"], s["v"], s["ks"], s["vs"]
        out = s["cache"].attend(q, s["batch"], scale=s["scale"], window=s["window"])
        return out if s["op"] == "attend" else (out, s["k"], s["v"], s["ks"], s["vs"])
    if s["op"] == "attend":
        return _attend_plain(s, s["q"])
    how = (s["positions"], s["freq"], s["mscale"], s["layout"], s["offset"], s["rot"], s["inverse"])
    if s["op"] == "rotate":
        return _rotated(s["x"], *how).to(s["dtype"])
    _append_plain(s)
    if s["op"] == "append":
        return s["k"], s["v"], s["ks"], s["vs"]
    return _attend_plain(s, _rotated(s["q"], *how).to(s["dtype"])), s["k"], s["v"], s["ks"], s["vs"]


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotate":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * es, "flops": 3 * n * case["rot"]}
    new, lens = _lengths(case)
    tokens = sum(new)
    dk, dv, kv = case["key_dim"], case["value_dim"], case["kv_heads"]
    b = f = 0
    if case["op"] != "attend":
        b += tokens * kv * (dk + dv) * (es + 1)
        f += tokens * kv * (3 * dk + 2 * (dk + dv))
    if case["op"] != "append":
        w, read, seen = case["window"], 0, 0
        for m, n in zip(new, lens):
            read += min(n, w + m - 1) if w else n
            short = max(0, min(m, w - (n - m) - 1)) if w else m   # the queries that see every token before them
            seen += short * (n - m) + short * (short + 1) // 2 + (m - short) * w
        b += read * kv * (dk + dv) + tokens * case["heads"] * (dk + dv) * es
        f += 2 * seen * case["heads"] * (dk + dv)
    return {"bytes": b, "flops": f}


# ---- the definition in 64 bits ------------------------------------------------------------------------------

def _exact_rotation(x, positions, freq, mscale, layout, offset, rot, inverse):
    x = x.double().clone()
    turn = torch.polar(torch.full((1,), mscale, dtype=torch.float64, device=x.device),
                       positions.double()[:, None] * freq * (-1 if inverse else 1))[:, None, :]
    first = torch.arange(rot // 2, device=x.device)
    i = first + offset if layout == "half" else 2 * first + offset
    j = i + rot // 2 if layout == "half" else i + 1
    z = torch.complex(x[..., i], x[..., j]) * turn
    x[..., i], x[..., j] = z.real, z.imag
    return x


def _exact_append(s):
    """Every value of the cache divided by its scale before it is rounded to 8 bits (old tokens: as they are)."""
    key = _exact_rotation(s["new_k"], s["positions"], s["freq"], s["mscale"], s["layout"], s["offset"], s["rot"], False)
    out = [s["k"].double(), s["v"].double(), s["ks"].double(), s["vs"].double()]
    start, lens, table = s["q_start"].tolist(), s["seq_lens"].tolist(), s["table"].tolist()
    for b, n in enumerate(lens):
        m = start[b + 1] - start[b]
        for blk in range((n - m) // BLOCK, -(-n // BLOCK)):
            lo, hi, base = max(n - m, blk * BLOCK), min(n, blk * BLOCK + BLOCK), blk * BLOCK
            page, at = table[b][blk // 4], blk % 4
            r0 = start[b] + lo - (n - m)
            o = at * BLOCK
            kn = key[r0:r0 + hi - lo].transpose(0, 1)                              # [H, t, D]
            vn = s["new_v"][r0:r0 + hi - lo].double().permute(1, 2, 0)             # [H, D, t]
            for rows, codes, scales, key_like in ((kn, out[0], out[2], True), (vn, out[1], out[3], False)):
                need = torch.exp2(torch.ceil(torch.log2(rows.abs().amax((1, 2)) / 448.0)))
                have = scales[page, :, at].clone()
                use = torch.maximum(need, have) if lo > base else need
                old = slice(o, o + lo - base)
                fresh = slice(o + lo - base, o + hi - base)
                u = use[:, None, None]
                if key_like:
                    codes[page, :, old] *= have[:, None, None] / u
                    codes[page, :, fresh] = rows / u
                else:
                    codes[page, :, :, old] *= have[:, None, None] / u
                    codes[page, :, :, fresh] = rows / u
                scales[page, :, at] = use
    return out


def _exact_attention(s, q, k, v, ks, vs):
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64, device=q.device)
    start, lens = s["q_start"].tolist(), s["seq_lens"].tolist()
    g = q.shape[1] // k.shape[1]
    for b, n in enumerate(lens):
        m = start[b + 1] - start[b]
        pages = s["table"][b, :-(-n // PAGE)].long()
        pos = torch.arange(n - m, n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)
        seen = j <= pos
        if s["window"]:
            seen &= pos - j < s["window"]
        for h in range(k.shape[1]):
            kh = (k[pages, h].double() * ks[pages, h].double().repeat_interleave(BLOCK, -1)[..., None]).flatten(0, 1)[:n]
            vh = (v[pages, h].double() * vs[pages, h].double().repeat_interleave(BLOCK, -1)[:, None, :])
            vh = vh.transpose(1, 2).flatten(0, 1)[:n]
            for i in range(h * g, h * g + g):
                x = (q[start[b]:start[b + 1], i].double() @ kh.T) * s["scale"]
                out[start[b]:start[b + 1], i] = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ vh
    return out


def exact(case, seed):
    if case["op"] == "append" and case["seqs"] * case["new"] > 60000:
        return None
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attention(s, s["q"], s["k"], s["v"], s["ks"], s["vs"])
    if case["op"] == "rotate":
        return _exact_rotation(s["x"], s["positions"], s["freq"], s["mscale"], s["layout"], s["offset"], s["rot"], s["inverse"])
    k, v, ks, vs = _exact_append(s)
    if case["op"] == "append":
        return k, v, ks, vs
    # the attention reads what the cache holds: the rounded values; its query is rounded to its type
    q = _exact_rotation(s["q"], s["positions"], s["freq"], s["mscale"], s["layout"], s["offset"], s["rot"], False)
    o = _exact_attention(s, q.to(s["dtype"]), k.to(E4M3), v.to(E4M3), ks, vs)
    return o, k, v, ks, vs
