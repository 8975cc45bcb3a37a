"""The 8-bit KV cache and the scoring of logits: what is measured of them.

Operators, each by its plain form (elementary torch operations in 32 bits,
the quantiser's border decisions in 64) and by the library's entry points:

  append    rows of K and V quantised into the cache as they are written,
            then read back (hs_kv8_append, hs_kv8_read)
  read      cached positions read back as floats (hs_kv8_read)
  attend    attention of query rows over the cache (hs_kv8_attend)
  logprobs  log probabilities of given tokens, entropy, rank and the top
            alternatives (hs_logprobs)

The cache: int8 codes with one f32 scale for each block of `block`
positions, each KV head, K and V apart. Shapes are those of the two models
that the benchmark runs (14 query and 2 KV heads of 64; 12 and 2 of 128;
151,936 tokens) and generic ones around them.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
VOCAB = 151936


def _kv(name, kind, dtype, n, m, ctx, nh, nkv, hd, block=1, layout=0, ragged=False):
    return dict(name=name, kind=kind, dtype=dtype, n=n, m=m, ctx=ctx, nh=nh, nkv=nkv, hd=hd, block=block,
                layout=layout, ragged=ragged)


def listed():
    return [
        # one decode step's rows of a 64-sequence batch, each at its own position
        _kv("append_b64_f32", "append", "f32", 64, 1, 1024, 14, 2, 64, ragged=True),
        # 16 prompts of 2,048 tokens entering the cache in one pass
        _kv("append_prompts_16x2048_bf16", "append", "bf16", 16, 2048, 2048, 12, 2, 128, block=32, layout=1),
        # a long sequence's layer read back whole (a hand-over to a worker with a cache of floats)
        _kv("read_ctx32768_f16", "read", "f16", 1, 32768, 32768, 12, 2, 128),
        # the same for a batch of sequences of different lengths
        _kv("read_b16_ragged_f32", "read", "f32", 16, 1500, 1500, 14, 2, 64, block=16, layout=1, ragged=True),
        # one chat turn: a single token over a short context
        _kv("attend_b1_ctx257_f32", "attend", "f32", 1, 1, 257, 14, 2, 64),
        # a decode step of the 64-sequence batch
        _kv("attend_b64_ctx2048_f32", "attend", "f32", 64, 1, 2048, 14, 2, 64, ragged=True),
        # a decode step of the 1.5B shape, in bf16, scales by blocks of 32
        _kv("attend_b16_ctx2560_bf16", "attend", "bf16", 16, 1, 2560, 12, 2, 128, block=32, layout=1, ragged=True),
        # a single token over a long context
        _kv("attend_b1_ctx32768_f16", "attend", "f16", 1, 1, 32768, 12, 2, 128, block=16),
        # four whole prompts of the 1.5B shape at once
        _kv("attend_prompts_4x2048_f32", "attend", "f32", 4, 2048, 2048, 12, 2, 128),
        # ragged prompt chunks behind cached positions
        _kv("attend_chunks_8x600_bf16", "attend", "bf16", 8, 600, 2047, 14, 2, 64, block=64, ragged=True),
        # the next token's alternatives in a chat turn
        dict(name="logprobs_1_f32", kind="logprobs", dtype="f32", rows=1, vocab=VOCAB, top=20, masked=True),
        # a whole prompt scored
        dict(name="logprobs_2048_bf16", kind="logprobs", dtype="bf16", rows=2048, vocab=VOCAB, top=5, masked=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "read", "attend", "attend", "logprobs"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "logprobs":
        vocab = _log(rng, 1000, VOCAB)
        rows = _log(rng, 1, max(1, min(2048, 2048 * VOCAB // vocab)))
        return dict(kind=kind, dtype=dtype, rows=rows if dtype == "bf16" else max(1, rows // 2), vocab=vocab,
                    top=rng.choice([0, 1, 5, 20, 33, 64]), masked=rng.random() < 0.5)
    nkv = rng.choice([1, 2, 4, 8])
    c = dict(kind=kind, dtype=dtype, nkv=nkv, nh=nkv * rng.choice([1, 3, 4, 6, 7, 8]), hd=rng.choice([64, 128]),
             block=rng.choice([1, 16, 32, 64, 128]), layout=rng.choice([0, 1]), ragged=rng.random() < 0.7)
    if kind == "attend" and rng.random() < 0.5:  # prompts and chunks of prompts
        m = _log(rng, 2, 2048)
        ctx = max(m, _log(rng, 16, 8192))
        n = max(1, min(64, _log(rng, 1, 16), 4 * 2048 * 2048 * 12 // (m * ctx * c["nh"])))
        if m * ctx * c["nh"] > 4 * 2048 * 2048 * 12:
            m = 4 * 2048 * 2048 * 12 // (ctx * c["nh"])
        return dict(c, n=n, m=m, ctx=ctx)
    if kind == "attend":  # single tokens
        ctx = _log(rng, 1, 32768)
        n = max(1, min(_log(rng, 1, 64), 131072 * 2 // (ctx * nkv)))
        return dict(c, n=n, m=1, ctx=ctx)
    m = rng.choice([1, _log(rng, 1, 8192)])
    n = max(1, min(_log(rng, 1, 64), 16 * 2048 * 2 // (m * nkv)))
    ctx = max(m, _log(rng, 1, 8192)) if kind == "append" else m
    return dict(c, n=n, m=m, ctx=ctx)


def _share(i, salt):
    """A fixed number in [0, 1) for sequence i."""
    return ((i * 2654435761 + salt * 40503 + 12345) * 2246822519 % 2**32) / 2**32


def _geometry(case):
    """Per sequence: positions cached once the rows are in, and rows. A ragged
    batch holds its longest sequence and shorter ones, down to a quarter."""
    lens, rows = [], []
    for i in range(case["n"]):
        part = 1.0 if not case["ragged"] or i == 0 else 0.25 + 0.75 * _share(i, 1)
        length = max(1, int(case["ctx"] * part))
        m = case["m"] if not case["ragged"] or i == 0 else max(1, int(case["m"] * (0.25 + 0.75 * _share(i, 2))))
        lens.append(length)
        rows.append(length if case["kind"] == "read" else min(m, length))
    return lens, rows


def work(case):
    b = BYTES[case["dtype"]]
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * b + case["rows"] * (16 + 8 * case["top"]), "flops": 4 * n}
    lens, rows = _geometry(case)
    nkv, nh, hd, block = case["nkv"], case["nh"], case["hd"], case["block"]
    r = sum(rows)
    scales = sum(-(-m // block) for m in rows) * nkv * 2 * 4
    if case["kind"] == "append":
        # rows in, codes and scales out; codes and scales in, rows out
        return {"bytes": 2 * r * nkv * hd * (b + 1) + scales + 2 * r * nkv * hd * (b + 1) + scales, "flops": 0}
    if case["kind"] == "read":
        return {"bytes": 2 * r * nkv * hd * (b + 1) + scales, "flops": 0}
    cached = sum(n * hd * 2 + -(-n // block) * 8 for n in lens) * nkv
    pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, rows))
    return {"bytes": cached + 2 * r * nh * hd * b, "flops": 4 * hd * nh * pairs}


def _quantise(x, old, old_scale, slot, pos, pos0, block):
    """Rows x [R, nkv, hd] at (slot, pos) into codes `old` [n, T, nkv, hd]
    (int8) and scales [n, blocks, nkv]; rows of one slot are consecutive from
    pos0[slot] on. Returns new codes and scales; the inputs stay."""
    n, t, nkv, hd = old.shape
    nb = old_scale.shape[1]
    at = slot * nb + pos // block
    top = torch.zeros(n * nb, nkv, device=x.device)
    top.scatter_reduce_(0, at[:, None].expand(-1, nkv), x.float().abs().amax(-1), "amax")
    touched = torch.zeros(n * nb, dtype=torch.bool, device=x.device)
    touched[at] = True
    touched = touched.view(n, nb, 1)
    need = (top / 127.0).view(n, nb, nkv)
    need = torch.where(need < 2.0**-126, torch.zeros_like(need), need)
    fresh = (torch.arange(nb, device=x.device) * block)[None, :, None] >= pos0[:, None, None]
    fresh = fresh | (old_scale == 0)
    mo, eo = torch.frexp(old_scale)
    mn, en = torch.frexp(need)
    grow = torch.where(fresh | (need == 0), torch.zeros_like(eo), (en - eo + (mn > mo).int()).clamp(min=0))
    scale = torch.where(touched, torch.where(fresh, need, torch.ldexp(old_scale, grow)), old_scale)
    grow = torch.where(touched, grow, torch.zeros_like(grow))
    per_pos = grow.repeat_interleave(block, dim=1)[:, :t, :, None]
    codes = torch.round(torch.ldexp(old.float(), -per_pos)).to(torch.int8)
    s = scale.view(n * nb, nkv)[at][:, :, None].double()
    c = torch.round(x.double() / torch.where(s == 0, torch.ones_like(s), s))
    codes.view(n * t, nkv, hd)[slot * t + pos] = torch.where(s == 0, torch.zeros_like(c), c).to(torch.int8)
    return codes, scale


def _keys(g, shape, nh, device):
    """Rows as a model's projections give them: a few wide channels in K."""
    x = torch.randn(shape, generator=g, device=device)
    wide = 1.0 + 5.0 * (torch.rand(shape[1:], generator=g, device=device) > 0.95).float()
    return x * wide


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case, "kind": case["kind"]}
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=g, device=dev)
        x = x.mul_(3.0).to(dt)
        if case["masked"]:  # the rows behind the tokenizer's last token
            x[:, vocab - vocab // 500 - 1:] = float("-inf")
        s["logits"] = x
        ids = torch.randint(0, vocab - vocab // 500 - 1, (rows,), generator=g, device=dev, dtype=torch.int32)
        s["ids"] = ids
        if own:
            s["out"] = dict(logp=torch.empty(rows, device=dev), entropy=torch.empty(rows, device=dev),
                            rank=torch.empty(rows, device=dev, dtype=torch.int32),
                            top_ids=torch.empty(rows, case["top"], device=dev, dtype=torch.int32),
                            top_logp=torch.empty(rows, case["top"], device=dev))
        return s
    lens, rows = _geometry(case)
    n, nkv, hd, block = case["n"], case["nkv"], case["hd"], case["block"]
    t = max(lens)
    nb = -(-t // block)
    s["rows"] = torch.tensor(rows, device=dev)
    s["pos0"] = torch.tensor([a - b for a, b in zip(lens, rows)], device=dev)
    # cached already: the positions before the rows that an append brings, else all of them
    have = [a - b for a, b in zip(lens, rows)] if case["kind"] == "append" else lens
    hslot, hpos = _places(torch.tensor(have, device=dev), torch.zeros(n, dtype=torch.long, device=dev))
    none = torch.zeros(n, dtype=torch.long, device=dev)
    hk = _keys(g, (sum(have), nkv, hd), case["nh"], dev).to(dt)
    hv = torch.randn((sum(have), nkv, hd), generator=g, device=dev).to(dt)
    s["slot"], s["pos"] = _places(s["rows"], s["pos0"])
    r = int(sum(rows))
    if case["kind"] == "append":
        s["k"] = _keys(g, (r, nkv, hd), case["nh"], dev).to(dt) * 1.25
        s["v"] = torch.randn((r, nkv, hd), generator=g, device=dev).to(dt) * 1.25
    elif case["kind"] == "attend":
        s["q"] = torch.randn((r, case["nh"], hd), generator=g, device=dev).to(dt)
    if own:
        import hotseat_b200 as hs
        spec = hs.KvSpec(1, nkv, hd, t, case["layout"])
        s["kvs"] = [hs.Kv.alloc8(spec, block=block) for _ in range(n)]
        s["set"] = hs.Kv8Set(s["kvs"], n_heads=case["nh"])
        if sum(have):
            s["set"].append(0, hk, hv, none.int(), _starts(torch.tensor(have, device=dev)))
        s["pos_d"], s["start_d"] = s["pos0"].int(), _starts(s["rows"]) if case["m"] > 1 else None
        if case["kind"] != "attend":
            s["out_k"] = torch.empty((r, nkv, hd), device=dev, dtype=dt)
            s["out_v"] = torch.empty((r, nkv, hd), device=dev, dtype=dt)
        else:
            s["out"] = torch.empty_like(s["q"])
        return s
    for name, x in (("k", hk), ("v", hv)):
        codes = torch.zeros(n, t, nkv, hd, dtype=torch.int8, device=dev)
        scale = torch.zeros(n, nb, nkv, device=dev)
        s["c" + name], s["s" + name] = _quantise(x, codes, scale, hslot, hpos, none, block) if sum(have) else (codes, scale)
    return s


def _starts(rows):
    return torch.cat([torch.zeros(1, dtype=torch.long, device=rows.device), rows.cumsum(0)]).int()


def _places(rows, pos0):
    """(slot, position) of every row of a ragged batch."""
    slot = torch.repeat_interleave(torch.arange(rows.numel(), device=rows.device), rows)
    first = rows.cumsum(0) - rows
    return slot, torch.arange(slot.numel(), device=rows.device) - first[slot] + pos0[slot]


def _values(codes, scale, block, slot=None, pos=None):
    """The values that codes stand for: all of them, or those of rows."""
    if slot is None:
        return codes.float() * scale.repeat_interleave(block, dim=1)[:, : codes.shape[1], :, None]
    return codes[slot, pos].float() * scale[slot, pos // block][:, :, None]


def run(s):
    case = s["case"]
    if s["kind"] == "logprobs":
        if own:
            import hotseat_b200 as hs
            o = s["out"]
            hs.logprobs(s["logits"], s["ids"], **o)
            return o
        return _plain_logprobs(s["logits"], s["ids"], case["top"])
    if s["kind"] == "append":
        if own:
            s["set"].append(0, s["k"], s["v"], s["pos_d"], s["start_d"])
            s["set"].read(0, s["out_k"], s["out_v"], s["pos_d"], s["start_d"])
            return {"k": s["out_k"], "v": s["out_v"]}
        out = {}
        for name in ("k", "v"):
            codes, scale = _quantise(s[name], s["c" + name], s["s" + name], s["slot"], s["pos"], s["pos0"],
                                     case["block"])
            out[name] = _values(codes, scale, case["block"], s["slot"], s["pos"]).to(s[name].dtype)
        return out
    if s["kind"] == "read":
        if own:
            s["set"].read(0, s["out_k"], s["out_v"], s["pos_d"], s["start_d"])
            return {"k": s["out_k"], "v": s["out_v"]}
        dt = DTYPES[case["dtype"]]
        return {name: _values(s["c" + name], s["s" + name], case["block"], s["slot"], s["pos"]).to(dt)
                for name in ("k", "v")}
    if own:
        s["set"].attend(0, s["q"], s["out"], s["pos_d"], s["start_d"])
        return s["out"]
    return _plain_attend(s["q"].float(), _values(s["ck"], s["sk"], case["block"]),
                         _values(s["cv"], s["sv"], case["block"]), s["slot"], s["pos"], s["pos0"],
                         case["m"]).to(s["q"].dtype)


def _plain_attend(q, k, v, slot, pos, pos0, m):
    """q [R, nh, hd] at (slot, pos) over k, v [n, T, nkv, hd], in q's type."""
    r, nh, hd = q.shape
    n, t, nkv, _ = k.shape
    qp = torch.zeros(n, m, nkv, nh // nkv, hd, dtype=q.dtype, device=q.device)
    row = pos - pos0[slot]
    qp[slot, row] = q.view(r, nkv, nh // nkv, hd)
    qp = qp.permute(0, 2, 3, 1, 4).reshape(n, nkv, nh // nkv * m, hd)
    x = torch.matmul(qp, k.permute(0, 2, 3, 1)).view(n, nkv, nh // nkv, m, t) * (1.0 / math.sqrt(hd))
    seen = torch.arange(t, device=q.device)[None, None, :] <= (pos0[:, None] + torch.arange(m, device=q.device))[:, :, None]
    x = x.masked_fill_(~seen[:, None, None], float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(n, nkv, nh // nkv * m, t), v.permute(0, 2, 1, 3)).view(n, nkv, nh // nkv, m, hd) / total
    return o.permute(0, 3, 1, 2, 4)[slot, row].reshape(r, nh, hd)


def _before(x, ids):
    """Each row's key of the order (value descending, id ascending), largest first."""
    b = (x + 0.0).view(torch.int32)
    b = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long()
    return (b << 32) + (2**32 - 1 - ids)


def _plain_logprobs(logits, ids, top):
    x = logits.float()
    t = ids.long()[:, None]
    m = x.amax(-1, keepdim=True)
    e = x - m
    p = e.exp()
    z = p.sum(-1, keepdim=True)
    logz = z.log()
    e = torch.where(p == 0, torch.zeros_like(e), e)
    entropy = (logz - (p * e).sum(-1, keepdim=True) / z)[:, 0]
    del e, p
    keys = _before(x, torch.arange(x.shape[1], device=x.device))
    rank = (keys > keys.gather(1, t)).sum(-1).int()
    best = keys.topk(top, dim=-1).values if top else keys[:, :0]
    best = 2**32 - 1 - (best & 0xFFFFFFFF)
    return dict(logp=(x.gather(1, t) - m - logz)[:, 0], entropy=entropy, rank=rank, top_ids=best.int(),
                top_logp=x.gather(1, best) - m - logz)


def exact(case, seed):
    """What run() returns, from the definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        parts = [_exact_scores(s["logits"][i:i + 64].double(), s["ids"][i:i + 64].long(), case["top"])
                 for i in range(0, case["rows"], 64)]
        return {k: torch.cat([p[k] for p in parts]) if parts[0][k] is not None else None for k in parts[0]}
    block = case["block"]
    lens, rows = _geometry(case)
    got = {"k": [], "v": []}
    outs = []
    at = 0
    for i, (length, m) in enumerate(zip(lens, rows)):
        p0 = length - m
        kv = []
        for name in ("k", "v"):
            codes, scale = s["c" + name][i].double(), s["s" + name][i].double()
            if case["kind"] == "append":
                x = s[name][at:at + m].double()
                vals = torch.empty_like(x)
                for b in range(p0 // block, (length - 1) // block + 1):
                    lo, hi = max(p0, b * block), min(length, (b + 1) * block)
                    part = x[lo - p0:hi - p0]
                    step = (part.abs().amax(dim=(0, 2)) / 127).float().double()  # a scale is held in 32 bits
                    if p0 > b * block:
                        held = scale[b]
                        times = torch.ceil(torch.log2(step / held)).clamp(min=0)
                        step = torch.where(held > 0, held * 2.0**times, step)
                    unit = torch.where(step > 0, step, torch.ones_like(step))[None, :, None]
                    vals[lo - p0:hi - p0] = torch.round(part / unit) * step[None, :, None]
                got[name].append(vals)
            else:
                kv.append(codes[:length] * scale.repeat_interleave(block, dim=0)[:length, :, None])
        if case["kind"] == "read":
            got["k"].append(kv[0])
            got["v"].append(kv[1])
        elif case["kind"] == "attend":
            q = s["q"][at:at + m].double().view(m, case["nkv"], -1, case["hd"])
            w = torch.einsum("mkgd,tkd->kgmt", q, kv[0]) / math.sqrt(case["hd"])
            hidden = torch.arange(length, device=w.device)[None, :] > p0 + torch.arange(m, device=w.device)[:, None]
            w = torch.softmax(w.masked_fill(hidden, float("-inf")), dim=-1)
            outs.append(torch.einsum("kgmt,tkd->mkgd", w, kv[1]).reshape(m, case["nh"], case["hd"]))
        at += m
    return torch.cat(outs) if outs else {k: torch.cat(v) for k, v in got.items()}


def _exact_scores(x, ids, top):
    logp = x - torch.logsumexp(x, dim=-1, keepdim=True)
    p = logp.exp()
    held = logp.gather(1, ids[:, None])[:, 0]
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    return dict(logp=held, entropy=entropy, rank=None, top_ids=None,
                top_logp=logp.topk(top, dim=-1).values if top else logp[:, :0])
