"""Mean negative log-likelihood over a token stream, the protocol of
hs-engine examples/ppl.rs (and llama-perplexity): independent windows of
`ctx` tokens, each decoded from position 0; only the second half of each
window is scored, so every scored token has at least ctx/2 tokens of
context behind it. A token's score is -log softmax(logits)[next] computed on
the device (hs_scratch_nll / hs_batch_nll: max-shifted, exp_f32, f64 sum).

    python -m hotseat_b200.ppl MODEL.gguf TEXT [ctx] [--numeric reference|fast|tc] [--ids] [--detail] [--kv8 BLOCK]

TEXT is tokenized by the model's own byte-level BPE (hotseat_b200.tok), or,
with --ids, read as whitespace-separated token ids. On the tensor-core path
the windows are decoded together as one batch, position by position. --detail
adds the mean entropy of the scored distributions and how often the token that
came was their first choice or among their first five (hs_*_logprobs); --kv8
keeps the cache in 8 bits, a scale per BLOCK positions (tensor-core path).
"""
import argparse
import math
import sys

import numpy as np

import hotseat_b200 as hs

NUMERIC = {"reference": hs.NUMERIC_REFERENCE, "fast": hs.NUMERIC_FAST, "tc": hs.NUMERIC_TC}


def score(model, ids, ctx=256, detail=False, kv8=0):
    """ppl.rs on `model` (a hs.Model loaded with max_ctx >= ctx) over token
    ids: returns tokens, windows, scored, mean_nll and ppl; with detail also
    mean_entropy (nats), top1 and top5 (shares of the scored tokens). kv8: an
    8-bit cache with a scale per that many positions (tensor-core models)."""
    ids = [int(t) for t in ids]
    chunks = len(ids) // ctx
    windows = [ids[c * ctx:(c + 1) * ctx] for c in range(chunks)]
    terms = [[] for _ in windows]  # per window, in position order
    more = []  # per scored token: entropy, rank
    kv_of = (lambda: model.kv8(block=kv8)) if kv8 else model.kv
    if model.cfg.numeric == hs.NUMERIC_TC:
        if windows:
            b = hs.Batch(model, len(windows))
            kvs = [kv_of() for _ in windows]
            for p in range(ctx):
                b.forward(kvs, [w[p] for w in windows], [p] * len(windows))
                if p >= ctx // 2 and p + 1 < ctx:
                    came = [w[p + 1] for w in windows]
                    for c, v in enumerate(b.nll(came)):
                        terms[c].append(float(v))
                    if detail:
                        o = b.logprobs(came)
                        more += zip(o["entropy"].tolist(), o["rank"].tolist())
            for kv in kvs:
                kv.close()
            b.close()
    else:
        kv, s = kv_of(), model.scratch()
        for c, w in enumerate(windows):
            for p, t in enumerate(w):
                model.forward(kv, t, p, s)
                if p >= ctx // 2 and p + 1 < len(w):
                    terms[c].append(s.nll(w[p + 1]))
                    if detail:
                        o = s.logprobs(w[p + 1])
                        more.append((float(o["entropy"]), int(o["rank"])))
        kv.close()
        s.close()
    nll = 0.0
    counted = 0
    for ws in terms:  # the reference's order: window by window, position by position
        for v in ws:
            nll += v
            counted += 1
    mean = nll / counted if counted else float("nan")
    r = {"tokens": len(ids), "windows": chunks, "ctx": ctx, "scored": counted, "mean_nll": mean,
         "ppl": math.exp(mean) if counted else float("nan")}
    if detail:
        n = len(more)
        r["mean_entropy"] = sum(e for e, _ in more) / n if n else float("nan")
        r["top1"] = sum(k < 1 for _, k in more) / n if n else float("nan")
        r["top5"] = sum(k < 5 for _, k in more) / n if n else float("nan")
    return r


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("model")
    ap.add_argument("text")
    ap.add_argument("ctx", nargs="?", type=int, default=256)
    ap.add_argument("--numeric", default="fast", choices=sorted(NUMERIC))
    ap.add_argument("--ids", action="store_true", help="TEXT holds token ids, not text")
    ap.add_argument("--detail", action="store_true", help="also mean entropy and how often the token was first, in the first five")
    ap.add_argument("--kv8", type=int, default=0, metavar="BLOCK", help="8-bit cache, a scale per BLOCK positions (tc)")
    ap.add_argument("--device", type=int, default=0)
    a = ap.parse_args(argv)
    raw = open(a.text, encoding="utf-8").read()
    if a.ids:
        ids = [int(x) for x in raw.split()]
    else:
        from hotseat_b200 import tok
        ids = tok.Tokenizer.from_gguf(a.model).encode(raw)
    m = hs.Model.load(a.model, max_ctx=a.ctx, device=a.device, numeric=NUMERIC[a.numeric])
    r = score(m, ids, a.ctx, detail=a.detail, kv8=a.kv8)
    print(f"tokens {r['tokens']} | windows {r['windows']} of {r['ctx']} | scored {r['scored']} | "
          f"mean NLL {r['mean_nll']:.5f} | ppl {r['ppl']:.5f}" +
          (f" | mean entropy {r['mean_entropy']:.5f} | first {r['top1']:.4f} | in the first five {r['top5']:.4f}"
           if a.detail else ""))
    return 0


if __name__ == "__main__":
    sys.exit(main())
