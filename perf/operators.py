"""The latent-attention operators of pb_b200 as measurable cases.

Four operators around one latent (MLA) cache, each with its plain form in
elementary torch operations and the call a user makes of the library:

  append   RMSNorm + RoPE of new tokens, the latent row quantised to 4 bits as
           it is written; the rotated query comes out in bf16
  read     rows of a 4-bit cache back as bf16 latent and key rows
  decode   absorbed attention of one new token a sequence over 4-bit caches
  prefill  causal attention of many new tokens a sequence over bf16 caches,
           in the expanded form

Shapes are the model's attention geometry: 16 heads (32 where a case says so),
nope 128, rope 64, latent 512, v 128. A 4-bit row is 512 codes of 4 bits
(stored code = 8 + q, q = rint(x / s) in -7..7, the even column in the low
nibble), one bf16 scale s = bf16(max|x| / 7) for each 64 columns, and the
rotated key part as 64 bf16 values: 400 bytes.
"""

import math

import torch

own = False

NOPE, ROPE, LATENT, VDIM, GROUP = 128, 64, 512, 128, 64
THETA, EPS = 10000.0, 1e-6
ROW_BYTES = LATENT // 2 + LATENT // GROUP * 2 + ROPE * 2
MAX_BATCH = 32


def listed():
    return [
        # one sequence's next token in a decode step: latency
        {"name": "append one token", "op": "append", "batch": 1, "tokens": 1, "rows": 4096, "heads": 16, "kv": "f32"},
        # a full decode batch, every sequence at its own position
        {"name": "append batch of 32", "op": "append", "batch": 32, "tokens": 32, "rows": 1024, "heads": 16, "kv": "f32"},
        # the prompts of three requests written into their caches (odd length)
        {"name": "append prompts", "op": "append", "batch": 3, "tokens": 8190, "rows": 4096, "heads": 16, "kv": "bf16"},
        # the context of one chunk, read back before its attention
        {"name": "read one context", "op": "read", "batch": 1, "rows": 2048, "ragged": False},
        # eight long contexts of different lengths read back
        {"name": "read long contexts", "op": "read", "batch": 8, "rows": 32768, "ragged": True},
        # one interactive sequence: few rows, latency
        {"name": "decode 1 x 4096", "op": "decode", "batch": 1, "rows": 4096, "heads": 16, "ragged": False, "q": "f32", "sharp": 1.0},
        # the long-context serving point
        {"name": "decode 8 x 32768", "op": "decode", "batch": 8, "rows": 32768, "heads": 16, "ragged": False, "q": "bf16", "sharp": 1.0},
        # a full batch of sequences of every age, with the peaked scores of trained heads
        {"name": "decode 32 ragged", "op": "decode", "batch": 32, "rows": 8192, "heads": 16, "ragged": True, "q": "f32", "sharp": 4.0},
        # a short follow-up message over a kept context
        {"name": "prefill 61 after 4035", "op": "prefill", "batch": 1, "tokens": 61, "context": 4035, "heads": 16, "ragged": False, "q": "bf16", "out": "bf16", "sharp": 1.0},
        # an ordinary prompt
        {"name": "prefill 2048", "op": "prefill", "batch": 1, "tokens": 2048, "context": 0, "heads": 16, "ragged": False, "q": "f32", "out": "bf16", "sharp": 1.0},
        # a long document
        {"name": "prefill 8192", "op": "prefill", "batch": 1, "tokens": 8192, "context": 0, "heads": 16, "ragged": False, "q": "bf16", "out": "bf16", "sharp": 4.0},
        # chunks of several requests, each with its own length and kept context
        {"name": "prefill 5 ragged chunks", "op": "prefill", "batch": 5, "tokens": 1024, "context": 2048, "heads": 16, "ragged": True, "q": "bf16", "out": "bf16", "sharp": 4.0},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "prefill"])
    if op == "append":
        batch = rng.randint(1, MAX_BATCH)
        tokens = max(batch, _spread(rng, 1, 8192))
        rows = max(16, tokens // batch + 1 + rng.randint(0, 512))
        return {"op": op, "batch": batch, "tokens": tokens, "rows": rows, "heads": rng.choice([16, 16, 32]),
                "kv": rng.choice(["f32", "bf16"])}
    if op == "read":
        batch = _spread(rng, 1, MAX_BATCH)
        return {"op": op, "batch": batch, "rows": _spread(rng, 1, 262144 // batch), "ragged": rng.random() < 0.7}
    if op == "decode":
        batch = _spread(rng, 1, MAX_BATCH)
        heads = rng.choice([16, 16, 32])
        return {"op": op, "batch": batch, "rows": _spread(rng, 1, 262144 * 16 // heads // batch), "heads": heads,
                "ragged": rng.random() < 0.7, "q": rng.choice(["f32", "bf16"]), "sharp": rng.choice([1.0, 4.0])}
    heads = rng.choice([16, 16, 32])
    pairs = 7680 * 4096 * 16 // heads  # attended pairs stay below the longest listed prompt's
    batch = _spread(rng, 1, 8)
    tokens = min(_spread(rng, 1, 8192 // batch), math.isqrt(2 * pairs // batch))
    context = rng.choice([0, _spread(rng, 1, max(1, min(16384 // batch, pairs // (batch * tokens) - tokens // 2)))])
    return {"op": op, "batch": batch, "tokens": tokens, "context": context, "heads": heads, "ragged": batch > 1 and rng.random() < 0.7,
            "q": rng.choice(["f32", "bf16"]), "out": "bf16", "sharp": rng.choice([1.0, 4.0])}


# ------------------------------------------------------------------ inputs
def _shape_rng():
    """Lengths belong to a case, not to a seed."""
    g = torch.Generator()
    g.manual_seed(1)
    return g


def _lens(n, top, ragged, g):
    """n lengths in 1..top, the longest exactly top; host data, as the calls take it."""
    if not ragged:
        return [top] * n
    u = torch.rand(n, generator=g).tolist()
    lens = [max(1, int(round(top ** v))) if k % 4 == 3 else max(1, int(top * v)) for k, v in enumerate(u)]
    lens[0] = top
    return lens


def _split_tokens(tokens, batch, rows, g):
    """Token counts of `batch` sequences: one each, or near-even shares of a prompt batch."""
    base = [tokens // batch + (1 if k < tokens % batch else 0) for k in range(batch)]
    for k in range(batch - 1):  # move some from one sequence to the next, within the caches
        move = min(int(torch.randint(0, base[k], (1,), generator=g)) // 4, rows - base[k + 1])
        base[k] -= move
        base[k + 1] += move
    return base


def _normal(shape, scale, dtype, g):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _quantise(x):
    """f32 latent rows [..., 512] -> (packed codes uint8 [..., 256], scales bf16 [..., 8])."""
    grp = x.reshape(*x.shape[:-1], LATENT // GROUP, GROUP)
    s = (grp.abs().amax(-1) / 7).to(torch.bfloat16)
    sf = s.float().unsqueeze(-1)
    q = torch.where(sf > 0, torch.round(grp / sf), torch.zeros_like(grp)).clamp(-7, 7)
    u = (q + 8).to(torch.uint8).reshape(x.shape)
    return u[..., 0::2] | (u[..., 1::2] << 4), s


def _dequantise(codes, scales):
    """f32 latent rows of packed codes and scales."""
    u = torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], LATENT)
    q = u.float() - 8
    return (q.reshape(*codes.shape[:-1], LATENT // GROUP, GROUP) * scales.float().unsqueeze(-1)).reshape(q.shape)


def _dtype(name):
    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


_engines = {}


def _engine():
    """The library context of the current device, as a serving process keeps one."""
    from pb_b200 import capi

    dev = torch.cuda.current_device()
    if dev not in _engines:
        _engines[dev] = capi.Context(dev)
    return capi, _engines[dev]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    hg = torch.Generator()
    hg.manual_seed(seed)
    lg = _shape_rng()
    op, batch = case["op"], case["batch"]
    st = {"case": case}
    if op == "append":
        counts = _split_tokens(case["tokens"], batch, case["rows"], lg) if case["tokens"] > batch else [1] * batch
        begins = [int(torch.randint(0, case["rows"] - n + 1, (1,), generator=hg)) for n in counts]
        seq = torch.repeat_interleave(torch.arange(batch), torch.tensor(counts))
        pos = torch.cat([torch.arange(b, b + n) for b, n in zip(begins, counts)])
        st["begins"], st["counts"] = begins, counts
        st["seq"], st["pos"] = seq.to("cuda", torch.int32), pos.to("cuda", torch.int32)
        t = len(pos)
        # projections of a normed hidden state, before the latent's own norm
        st["kv"] = _normal((t, LATENT + ROPE), 1.5, _dtype(case["kv"]), g)
        st["query"] = _normal((t, case["heads"], NOPE + ROPE), 1.0, torch.float32, g)
        st["norm"] = 1 + 0.1 * torch.randn(LATENT, generator=g, device="cuda")
        rows = case["rows"]
        st["codes"] = torch.zeros(batch, rows, LATENT // 2, dtype=torch.uint8, device="cuda")
        st["scales"] = torch.zeros(batch, rows, LATENT // GROUP, dtype=torch.bfloat16, device="cuda")
        st["k_rope"] = torch.zeros(batch, rows, ROPE, dtype=torch.bfloat16, device="cuda")
        st["query_out"] = torch.empty(t, case["heads"], NOPE + ROPE, dtype=torch.bfloat16, device="cuda")
        st["latent_out"] = torch.empty(t, LATENT, dtype=torch.bfloat16, device="cuda")
        st["key_out"] = torch.empty(t, ROPE, dtype=torch.bfloat16, device="cuda")
    elif op in ("read", "decode"):
        rows = case["rows"]
        st["lens"] = _lens(batch, rows, case["ragged"], lg)
        codes, scales = [], []
        for _ in range(batch):  # one sequence at a time: the f32 rows are large
            c, s = _quantise(_normal((rows, LATENT), 1.0, torch.float32, g))
            codes.append(c)
            scales.append(s)
        st["codes"], st["scales"] = torch.stack(codes), torch.stack(scales)
        st["k_rope"] = _normal((batch, rows, ROPE), 1.0, torch.bfloat16, g)
        if op == "read":
            total = sum(st["lens"])
            st["latent_out"] = torch.empty(total, LATENT, dtype=torch.bfloat16, device="cuda")
            st["key_out"] = torch.empty(total, ROPE, dtype=torch.bfloat16, device="cuda")
        else:
            st["query"] = _normal((batch, case["heads"], NOPE + ROPE), case["sharp"], _dtype(case["q"]), g)
            st["out"] = torch.empty(batch, case["heads"], VDIM, dtype=torch.bfloat16, device="cuda")
    else:
        q_lens = _lens(batch, case["tokens"], case["ragged"], lg)
        ctx = _lens(batch, case["context"], case["ragged"], lg) if case["context"] else [0] * batch
        ctx = ctx[::-1]  # the longest chunk does not have the longest context
        st["q_lens"], st["lens"] = q_lens, [a + b for a, b in zip(q_lens, ctx)]
        st["c_kv"] = [_normal((n, LATENT), 1.0, torch.bfloat16, g) for n in st["lens"]]
        st["k_rope"] = [_normal((n, ROPE), 1.0, torch.bfloat16, g) for n in st["lens"]]
        t = sum(q_lens)
        st["query"] = _normal((t, case["heads"], NOPE + ROPE), case["sharp"], _dtype(case["q"]), g)
        st["out"] = torch.empty(t, case["heads"], VDIM, dtype=_dtype(case["out"]), device="cuda")
    if op in ("decode", "prefill"):
        st["w_uk"] = _normal((case["heads"], NOPE, LATENT), 0.02, torch.bfloat16, g)
        st["w_uv"] = _normal((case["heads"], VDIM, LATENT), 0.02, torch.bfloat16, g)
    if own:
        capi, ctx = _engine()
        st["ctx"], st["config"] = ctx, capi.mla_config(heads=case.get("heads", 16))
        if op != "prefill":
            st["cache"] = capi.MlaQ4Cache(list(st["codes"]), list(st["scales"]), list(st["k_rope"]))
        if op == "append":
            ctx.rope_reserve(65536, ROPE, THETA)
            if case["tokens"] == batch:
                st["seq"] = None  # token i is sequence i's
        if op == "decode":
            ctx.mla_q4_reserve(st["config"], batch)
        if op == "prefill":
            ctx.mla_prefill_reserve(st["config"], q_lens, st["lens"])
            st["kept"] = capi.MlaCache(st["c_kv"], st["k_rope"])
    return st


# ------------------------------------------------------------------ plain forms
def _rotate(x, pos):
    """RoPE of the last 64 values (interleaved pairs -> split halves), f32; angles in 64 bits."""
    ang = pos.double().unsqueeze(-1) * THETA ** (-torch.arange(0, ROPE, 2, device=x.device).double() / ROPE)
    c, s = ang.cos().float(), ang.sin().float()
    while c.dim() < x.dim():
        c, s = c.unsqueeze(1), s.unsqueeze(1)
    x0, x1 = x[..., 0::2], x[..., 1::2]
    return torch.cat((x0 * c - x1 * s, x1 * c + x0 * s), -1)


def _plain_append(st):
    kv, pos, seq = st["kv"].float(), st["pos"].long(), st["seq"].long()
    lat = kv[:, :LATENT]
    # the mean square in 64 bits: a code next to a border depends on its last bit
    scale = (1 / torch.sqrt(lat.double().square().mean(-1, keepdim=True) + EPS)).float()
    codes, scales = _quantise(lat * scale * st["norm"])
    st["codes"][seq, pos] = codes
    st["scales"][seq, pos] = scales
    st["k_rope"][seq, pos] = _rotate(kv[:, LATENT:], pos).to(torch.bfloat16)
    q = torch.cat((st["query"][..., :NOPE], _rotate(st["query"][..., NOPE:], pos)), -1).to(torch.bfloat16)
    lat = _dequantise(st["codes"][seq, pos], st["scales"][seq, pos]).to(torch.bfloat16)
    return q, lat, st["k_rope"][seq, pos]


def _kept(st):
    """Mask [batch, rows] of the rows that each sequence has."""
    rows = torch.arange(st["codes"].shape[1], device="cuda")
    return rows < torch.tensor(st["lens"], device="cuda").unsqueeze(1)


def _plain_read(st):
    kept = _kept(st)
    return _dequantise(st["codes"][kept], st["scales"][kept]).to(torch.bfloat16), st["k_rope"][kept]


def _softmax(s):
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_decode(st):
    lat = _dequantise(st["codes"], st["scales"])  # [B, L, 512] f32
    q = st["query"].float()
    q_lat = torch.einsum("bhd,hdc->bhc", q[..., :NOPE], st["w_uk"].float())
    s = torch.matmul(q_lat, lat.transpose(1, 2)) + torch.matmul(q[..., NOPE:], st["k_rope"].float().transpose(1, 2))
    s = (s / math.sqrt(NOPE + ROPE)).masked_fill(~_kept(st).unsqueeze(1), -math.inf)
    ctx = torch.matmul(_softmax(s), lat)
    return torch.einsum("bhc,hdc->bhd", ctx, st["w_uv"].float()).to(torch.bfloat16)


def _plain_prefill(st):
    lens, q_lens = torch.tensor(st["lens"], device="cuda"), torch.tensor(st["q_lens"], device="cuda")
    pad = torch.nn.utils.rnn.pad_sequence
    c = pad(st["c_kv"], batch_first=True).float()  # [B, L, 512]
    kr = pad(st["k_rope"], batch_first=True).float()
    q = pad(list(torch.split(st["query"], st["q_lens"])), batch_first=True).float()  # [B, T, H, 192]
    k = torch.einsum("blc,hdc->bhld", c, st["w_uk"].float())
    v = torch.einsum("blc,hdc->bhld", c, st["w_uv"].float())
    s = torch.einsum("bthd,bhld->bhtl", q[..., :NOPE], k)
    s += torch.einsum("bthd,bld->bhtl", q[..., NOPE:], kr)
    s /= math.sqrt(NOPE + ROPE)
    row = torch.arange(q.shape[1], device="cuda")
    last = (lens - q_lens).unsqueeze(1) + row  # [B, T]: the last key a token sees
    s.masked_fill_((torch.arange(c.shape[1], device="cuda") > last.unsqueeze(-1)).unsqueeze(1), -math.inf)
    o = torch.einsum("bhtl,bhld->bthd", _softmax(s), v)
    return o[row < q_lens.unsqueeze(1)].to(st["out"].dtype)


def run(st):
    op = st["case"]["op"]
    if not own:
        return {"append": _plain_append, "read": _plain_read, "decode": _plain_decode, "prefill": _plain_prefill}[op](st)
    ctx, cfg = st["ctx"], st["config"]
    if op == "append":
        ctx.mla_q4_append(cfg, st["kv"], st["pos"], st["cache"], sequences=st["seq"], query=st["query"],
                          query_out=st["query_out"], latent_norm=st["norm"], eps=EPS)
        ctx.mla_q4_read(cfg, st["cache"], st["begins"], st["counts"], st["latent_out"], st["key_out"])
        return st["query_out"], st["latent_out"], st["key_out"]
    if op == "read":
        ctx.mla_q4_read(cfg, st["cache"], None, st["lens"], st["latent_out"], st["key_out"])
        return st["latent_out"], st["key_out"]
    if op == "decode":
        ctx.mla_q4_decode(cfg, st["query"], st["cache"], st["lens"], st["w_uk"], st["w_uv"], st["out"])
        return st["out"]
    ctx.mla_prefill(cfg, st["query"], st["q_lens"], st["kept"], st["lens"], st["w_uk"], st["w_uv"], st["out"])
    return st["out"]


# ------------------------------------------------------------------ work
def work(case):
    op, heads = case["op"], case.get("heads", 16)
    g = _shape_rng()
    weights = heads * (NOPE + VDIM) * LATENT * 2
    if op == "append":
        t = case["tokens"]
        kv = (LATENT + ROPE) * (4 if case["kv"] == "f32" else 2)
        return {"bytes": t * (kv + heads * (NOPE + ROPE) * (4 + 2) + ROW_BYTES + (LATENT + ROPE) * 2), "flops": t * 10 * (LATENT + (heads + 1) * ROPE)}
    if op == "read":
        n = sum(_lens(case["batch"], case["rows"], case["ragged"], g))
        return {"bytes": n * (ROW_BYTES + (LATENT + ROPE) * 2), "flops": n * LATENT}
    if op == "decode":
        n, b = sum(_lens(case["batch"], case["rows"], case["ragged"], g)), case["batch"]
        io = b * heads * ((NOPE + ROPE) * (4 if case["q"] == "f32" else 2) + VDIM * 2)
        return {"bytes": n * ROW_BYTES + weights + io,
                "flops": 2 * heads * (n * (2 * LATENT + ROPE) + b * (NOPE + VDIM) * LATENT)}
    q_lens = _lens(case["batch"], case["tokens"], case["ragged"], g)
    ctx = (_lens(case["batch"], case["context"], case["ragged"], g) if case["context"] else [0] * case["batch"])[::-1]
    t, n = sum(q_lens), sum(q_lens) + sum(ctx)
    pairs = sum(q * c + q * (q + 1) // 2 for q, c in zip(q_lens, ctx))
    expanded = 2 * heads * (pairs * (NOPE + ROPE + VDIM) + n * LATENT * (NOPE + VDIM))
    absorbed = 2 * heads * (pairs * (2 * LATENT + ROPE) + t * LATENT * (NOPE + VDIM))
    io = t * heads * ((NOPE + ROPE) * (4 if case["q"] == "f32" else 2) + VDIM * (2 if case["out"] == "bf16" else 4))
    return {"bytes": n * (LATENT + ROPE) * 2 + weights + io, "flops": min(expanded, absorbed)}


# ------------------------------------------------------------------ 64 bits
def _codes64(st, b, begin, end):
    """(q, s) of rows [begin, end) of sequence b, as 64-bit values."""
    raw = st["codes"][b, begin:end]
    q = torch.empty(end - begin, LATENT, dtype=torch.float64, device="cuda")
    q[:, 0::2] = (raw % 16).double()
    q[:, 1::2] = (raw // 16).double()
    return q - 8, st["scales"][b, begin:end].double()


def _latent64(st, b, begin, end):
    q, s = _codes64(st, b, begin, end)
    for j in range(LATENT // GROUP):
        q[:, j * GROUP:(j + 1) * GROUP] *= s[:, j:j + 1]
    return q


def _rope64(x, pos):
    out = torch.empty_like(x)
    for p in range(ROPE // 2):
        a = pos.double() * THETA ** (-2.0 * p / ROPE)
        a = a.reshape(-1, *[1] * (x.dim() - 2))
        out[..., p] = x[..., 2 * p] * torch.cos(a) - x[..., 2 * p + 1] * torch.sin(a)
        out[..., ROPE // 2 + p] = x[..., 2 * p + 1] * torch.cos(a) + x[..., 2 * p] * torch.sin(a)
    return out


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    if op == "append":
        kv, pos = st["kv"].double(), st["pos"]
        x = kv[:, :LATENT]
        x = x / torch.sqrt((x * x).sum(1, keepdim=True) / LATENT + EPS) * st["norm"].double()
        lat = torch.empty_like(x)
        for j in range(LATENT // GROUP):
            c = x[:, j * GROUP:(j + 1) * GROUP]
            s = (c.abs().max(1, keepdim=True).values / 7).to(torch.bfloat16).double()
            lat[:, j * GROUP:(j + 1) * GROUP] = torch.round(c / s) * s
        q = st["query"].double()
        q = torch.cat((q[..., :NOPE], _rope64(q[..., NOPE:], pos)), -1)
        return q, lat, _rope64(kv[:, LATENT:], pos)
    if op == "read":
        lat = [_latent64(st, b, 0, n) for b, n in enumerate(st["lens"])]
        return torch.cat(lat), torch.cat([st["k_rope"][b, :n].double() for b, n in enumerate(st["lens"])])
    heads, scale = case["heads"], 1 / math.sqrt(NOPE + ROPE)
    wk, wv = st["w_uk"].double(), st["w_uv"].double()
    if op == "decode":
        out = torch.empty(case["batch"], heads, VDIM, dtype=torch.float64, device="cuda")
        for b, n in enumerate(st["lens"]):
            c, kr, q = _latent64(st, b, 0, n), st["k_rope"][b, :n].double(), st["query"][b].double()
            ql = (q[:, :NOPE].unsqueeze(1) @ wk).squeeze(1)
            p = torch.softmax((ql @ c.T + q[:, NOPE:] @ kr.T) * scale, -1)
            out[b] = (wv @ (p @ c).unsqueeze(-1)).squeeze(-1)
        return out
    outs, at = [], 0
    for b, (t, n) in enumerate(zip(st["q_lens"], st["lens"])):
        c, kr = st["c_kv"][b].double(), st["k_rope"][b].double()
        q = st["query"][at:at + t].double()
        at += t
        out = torch.empty(t, heads, VDIM, dtype=torch.float64, device="cuda")
        hidden = torch.ones(t, n, dtype=torch.bool, device="cuda").triu(n - t + 1)
        for h in range(heads):
            key = torch.cat((c @ wk[h].T, kr), 1)
            s = (q[:, h] @ key.T * scale).masked_fill(hidden, -math.inf)
            out[:, h] = torch.softmax(s, -1) @ (c @ wv[h].T)
        outs.append(out)
    return torch.cat(outs)
