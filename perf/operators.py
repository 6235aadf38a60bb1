"""What the preference-tuning and 8-bit operators are measured on: cases, their inputs, plain forms, the library's calls and the results in 64 bits.

Kinds of cases
  score   log-probabilities of given tokens under a batch of logits and their sums per sequence (a frozen model scores finished summaries)
  pref    paired preference loss on the logits of [chosen; rejected] summaries, with the gradient of the logits
  policy  clipped policy loss with a KL term on the logits of sampled summaries, with the gradient of the logits
  embed   embedding lookup with scaling, and the gradient of the table
  i8      y = x W^T (+ bias, GELU) with 8-bit weights scaled per output channel and activations quantised per token inside the call

`own` False: `run` computes the plain form in elementary torch operations; True: it calls the library.
"""
import math

import numpy as np
import torch

own = False

VOCAB, PITCH, WIDTH, FFN = 50265, 50304, 1024, 4096            # cfg/bart-large.json; PITCH = the row pitch of the framework's logits buffers
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ES = {"f32": 4, "bf16": 2}


def listed():
    return [
        # four hypotheses' next tokens under the frozen model, f32 logits of the decode step: latency
        dict(name="score-4x1-f32", kind="score", N=4, T=1, V=VOCAB, pitch=PITCH, dt="f32", average=False, empty=False, banned=False),
        # 72 reviews of up to 141 tokens, logits packed without padding columns (rows start at any even byte)
        dict(name="score-72x141-bf16", kind="score", N=72, T=141, V=VOCAB, pitch=VOCAB, dt="bf16", average=True, empty=True, banned=False),
        # a single pair at a small vocabulary: the smallest training call
        dict(name="pref-1x33-v1009-f32", kind="pref", N=2, T=33, V=1009, pitch=1009, dt="f32", beta=0.1, smoothing=0.1, average=True, empty=False, banned=False),
        # 36 pairs of 128-token summaries: one device's step
        dict(name="pref-36x128-bf16", kind="pref", N=72, T=128, V=VOCAB, pitch=PITCH, dt="bf16", beta=0.1, smoothing=0.0, average=False, empty=False, banned=False),
        # three sampled summaries, f32 logits, no reference model, an odd length
        dict(name="policy-3x57-f32", kind="policy", N=3, T=57, V=VOCAB, pitch=VOCAB, dt="f32", low=0.2, high=0.2, kl=0.0, reduction="sequence", empty=False, banned=False),
        # 72 sampled summaries of 128 tokens with the KL term: one device's step
        dict(name="policy-72x128-bf16", kind="policy", N=72, T=128, V=VOCAB, pitch=PITCH, dt="bf16", low=0.2, high=0.28, kl=0.05, reduction="token", empty=True, banned=True),
        # one short sentence on a small table: latency
        dict(name="embed-1x21-v1009-f32", kind="embed", N=1, T=21, V=1009, D=256, dt="f32", scale=16.0),
        # the per-device batch of one business: nine reviews of 128 tokens
        dict(name="embed-9x128-bf16", kind="embed", N=9, T=128, V=VOCAB, D=WIDTH, dt="bf16", scale=32.0),
        # the benchmark's batch: 128 businesses of nine reviews
        dict(name="embed-1152x128-bf16", kind="embed", N=1152, T=128, V=VOCAB, D=WIDTH, dt="bf16", scale=32.0),
        # a decode step's projection: two businesses of four beams
        dict(name="i8-8x1024x1024-bf16", kind="i8", M=8, N=WIDTH, K=WIDTH, dt="bf16", out="bf16", bias=True, gelu=False),
        # the decode step's vocabulary projection, eight businesses of four beams
        dict(name="i8-32x50265x1024-bf16", kind="i8", M=32, N=VOCAB, K=WIDTH, dt="bf16", out="f32", bias=False, gelu=False),
        # the frozen model's feed-forward up-projection over 288 summaries of 128 tokens
        dict(name="i8-36864x4096x1024-bf16", kind="i8", M=36864, N=FFN, K=WIDTH, dt="bf16", out="bf16", bias=True, gelu=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["score", "pref", "policy", "embed", "i8"])
    dt = rng.choice(["f32", "bf16"])
    if kind == "embed":
        c = dict(kind=kind, N=_log(rng, 1, 1152), T=_log(rng, 1, 224), V=_log(rng, 64, VOCAB), D=rng.choice([64, 100, 250, 256, 512, 777, WIDTH]), dt=dt,
                 scale=rng.choice([1.0, 16.0, 32.0]))
        c["N"] = max(1, min(c["N"], 1152 * 128 * 2 // (c["T"] * ES[dt])))
        return c
    if kind == "i8":
        M, N, K = _log(rng, 1, 36864), _log(rng, 17, VOCAB), rng.choice([_log(rng, 16, FFN), WIDTH, FFN])
        M = max(1, min(M, 36864 * FFN * WIDTH // (N * K), 36864 * FFN // N))
        return dict(kind=kind, M=M, N=N, K=K, dt=dt, out=rng.choice(["f32", "bf16"]) if M * N <= 36864 * 2048 else "bf16", bias=rng.random() < 0.6, gelu=rng.random() < 0.3)
    V = rng.choice([VOCAB, _log(rng, 64, VOCAB)])
    T = _log(rng, 1, 224)
    N = 2 * _log(rng, 1, 36)
    N = max(2, min(N, 72 * 128 * PITCH * 2 // (T * (V + 128) * ES[dt]) // 2 * 2))
    c = dict(kind=kind, N=N, T=T, V=V, pitch=rng.choice([V, (V + 127) // 128 * 128]), dt=dt, empty=rng.random() < 0.3, banned=rng.random() < 0.3)
    if kind == "score":
        c.update(average=rng.random() < 0.5)
    elif kind == "pref":
        c.update(beta=rng.choice([0.05, 0.1, 0.5]), smoothing=rng.choice([0.0, 0.1]), average=rng.random() < 0.5)
    else:
        c.update(low=0.2, high=rng.choice([0.2, 0.28]), kl=rng.choice([0.0, 0.05]), reduction=rng.choice(["token", "sequence"]))
    return c


def _lengths(c):
    """Counted tokens of every sequence: ragged, all of them in the first sequence, none in the second where `empty` is set."""
    ln = [c["T"] - (5 * i) % (c["T"] // 3 + 1) for i in range(c["N"])]
    if c.get("empty") and c["N"] > 2:
        ln[1] = 0
    return ln


def _token_p(V):
    """Rank-frequency weights of natural text over the ids behind the four special ones."""
    p = np.zeros(V)
    p[4:] = 1.0 / (np.arange(V - 4) + 2.7)
    return p / p.sum()


def work(case):
    c = case
    k = c["kind"]
    if k == "i8":
        return {"bytes": c["M"] * c["K"] * ES[c["dt"]] + c["N"] * (c["K"] + 4) + c["M"] * c["N"] * ES[c["out"]] + (4 * c["N"] if c["bias"] else 0),
                "flops": 2 * c["M"] * c["N"] * c["K"]}
    rows = sum(_lengths(c))
    if k == "embed":
        es, n = ES[c["dt"]], c["N"] * c["T"]
        distinct = float((1.0 - (1.0 - _token_p(c["V"])) ** rows).sum())
        return {"bytes": int(distinct * c["D"] * es) + 8 * n + 2 * n * c["D"] * es + 4 * c["V"] * c["D"], "flops": 2 * n * c["D"]}
    read = rows * c["V"] * ES[c["dt"]]
    R = c["N"] * c["T"]
    if k == "score":
        return {"bytes": read + 12 * R + 4 * c["N"], "flops": 4 * rows * c["V"]}
    return {"bytes": read + R * c["V"] * ES[c["dt"]] + 24 * R, "flops": 8 * rows * c["V"]}


# ---------------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1234567 + 977 * int(seed))
    return g


def _quantize(x):
    """Per-row symmetric 8-bit values and scales: q = 127 x / max |x| rounded to the nearest, ties to even; scale = max |x| / 127 in f32."""
    x = x.float()
    top = x.abs().amax(1)
    q = torch.where(top[:, None] > 0, torch.round(x * 127.0 / top[:, None]), torch.zeros_like(x))
    return q, top / 127.0


def _inputs(c, seed):
    """What every form of a case starts from (tensors on the device)."""
    g, dev = _gen(seed), "cuda"

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if c["kind"] == "i8":
        x = randn(c["M"], c["K"]) * (0.5 + torch.rand(c["M"], 1, generator=g, device=dev))
        x[:, :: max(1, c["K"] // 7)] *= 4.0                                    # a few channels carry most of a token's range
        w = randn(c["N"], c["K"]) * 0.02
        return dict(x=x.to(DT[c["dt"]]), w=w.to(torch.bfloat16), bias=randn(c["N"]) * 0.1 if c["bias"] else None)
    ln = torch.tensor(_lengths(c), device=dev)
    pos = torch.arange(c["T"], device=dev)
    keep = pos[None, :] < ln[:, None]
    if c["kind"] == "embed":
        p = torch.tensor(_token_p(c["V"]), device=dev)
        u = torch.rand(c["N"], c["T"], generator=g, device=dev, dtype=torch.float64)
        ids = torch.searchsorted(torch.cumsum(p, 0), u).clamp(4, c["V"] - 1)
        ids = torch.where(keep, ids, torch.ones_like(ids))                      # padding id 1
        return dict(ids=ids, table=(randn(c["V"], c["D"]) * 0.02).to(DT[c["dt"]]), dy=(randn(c["N"], c["T"], c["D"]) * 0.01).to(DT[c["dt"]]))
    N, T, V = c["N"], c["T"], c["V"]
    labels = torch.randint(0, V, (N, T), generator=g, device=dev)
    buf = torch.empty(N, T, c["pitch"], dtype=DT[c["dt"]], device=dev)
    for n in range(N):                                                          # a sequence at a time: no f32 copy of the whole batch
        x = randn(T, c["pitch"]) * 2.0
        x[pos, labels[n]] += 6.0                                                # a model that gives its own tokens a fair share
        if c["banned"]:
            x[:, 7 % V] = float("-inf")                                         # a suppressed token
            x[pos, labels[n]] = torch.where(labels[n] == 7 % V, torch.zeros_like(x[:, 0]), x[pos, labels[n]])
        buf[n] = x.to(buf.dtype)
    d = dict(logits=buf[:, :, :V], labels=torch.where(keep, labels, torch.full_like(labels, -100)))
    if c["kind"] == "pref":
        d["ref"] = -T * 0.5 - torch.rand(N, generator=g, device=dev) * 4.0
        if c["average"]:
            d["ref"] = d["ref"] / T
    elif c["kind"] == "policy":
        lp = torch.stack([torch.log_softmax(buf[n, :, :V].float(), -1).gather(-1, labels[n][:, None])[:, 0] for n in range(N)])
        step = randn(N, T) * 0.2
        near = ((step.exp() - (1 + c["high"])).abs() < 4e-3) | ((step.exp() - (1 - c["low"])).abs() < 4e-3)
        step = torch.where(near, torch.zeros_like(step), step)
        zero = torch.zeros_like(lp)
        d["old"] = torch.where(keep, lp - step, zero)
        d["ref"] = torch.where(keep, lp + randn(N, T) * 0.3, zero) if c["kl"] else None
        d["adv"] = randn(N)                                                     # one advantage for each summary
    return d


def prepare(case, seed):
    st = dict(case=case, **_inputs(case, seed))
    if case["kind"] == "i8":
        if own:
            from multimodalsum_amd import Int8Linear
            st["linear"] = Int8Linear(st["w"], st["bias"], gelu=case["gelu"], out_dtype=DT[case["out"]])
        else:
            st["wq"], st["ws"] = _quantize(st["w"])
            st["wq"] = st["wq"].to(torch.int8)
        del st["w"]
    return st


# ---------------------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    import multimodalsum_amd as mm
    c = s["case"]
    if c["kind"] == "score":
        seq, tok = mm.sequence_logprobs(s["logits"], s["labels"], average=c["average"])
        return {"sequence": seq, "token": tok}
    if c["kind"] == "pref":
        loss, margins, dlogits = mm.preference_loss_and_grad(s["logits"], s["labels"], s["ref"], beta=c["beta"], label_smoothing=c["smoothing"], average=c["average"])
        return {"loss": loss, "margins": margins, "dlogits": dlogits}
    if c["kind"] == "policy":
        loss, kl, clipped, tok, dlogits = mm.policy_loss_and_grad(s["logits"], s["labels"], s["old"], s["adv"], s["ref"], clip_low=c["low"], clip_high=c["high"],
                                                                  kl_coef=c["kl"], reduction=c["reduction"])
        return {"loss": loss, "kl": kl, "clipped": clipped, "token": tok, "dlogits": dlogits}
    if c["kind"] == "embed":
        y = mm.scaled_embedding(s["ids"], s["table"], c["scale"])
        return {"y": y, "dtable": mm.scaled_embedding_grad(s["dy"], s["ids"], c["V"], c["scale"], padding_idx=1)}
    return s["linear"](s["x"])


def _plain_logprobs(x, labels):
    keep = (labels >= 0) & (labels < x.shape[-1])
    lab = torch.where(keep, labels, torch.zeros_like(labels))
    m = x.amax(-1, keepdim=True)
    z = torch.exp(x - m)
    total = z.sum(-1, keepdim=True)
    lp = (x.gather(-1, lab[..., None]) - m - torch.log(total))[..., 0]
    return keep, lab, torch.where(keep, lp, torch.zeros_like(lp)), z / total


def _plain_dlogits(p, lab, coef, dtype):
    d = p * -coef[..., None]
    d.scatter_add_(-1, lab[..., None], coef[..., None])
    return d.to(dtype)


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "i8":
        q, sx = _quantize(s["x"])
        y = (q @ s["wq"].float().t()) * sx[:, None] * s["ws"][None, :]
        if s["bias"] is not None:
            y = y + s["bias"]
        if c["gelu"]:
            y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
        return y.to(DT[c["out"]])
    if c["kind"] == "embed":
        ids = s["ids"].reshape(-1)
        y = (s["table"][ids].float() * c["scale"]).to(s["table"].dtype).reshape(c["N"], c["T"], c["D"])
        dt = torch.zeros(c["V"], c["D"], device=ids.device)
        dt.index_add_(0, ids, s["dy"].reshape(-1, c["D"]).float())
        dt *= c["scale"]
        dt[1] = 0.0
        return {"y": y, "dtable": dt}
    keep, lab, lp, p = _plain_logprobs(s["logits"].float(), s["labels"])
    cnt = keep.sum(1).clamp(min=1).float()
    if c["kind"] == "score":
        seq = lp.sum(1)
        return {"sequence": seq / cnt if c["average"] else seq, "token": lp}
    if c["kind"] == "pref":
        seq = lp.sum(1) / cnt if c["average"] else lp.sum(1)
        P, e = c["N"] // 2, c["smoothing"]
        r = seq - s["ref"]
        h = c["beta"] * (r[:P] - r[P:])
        soft_neg, soft_pos = _softplus(-h), _softplus(h)
        loss = ((1 - e) * soft_neg + e * soft_pos).mean()
        dh = (e - torch.sigmoid(-h)) * c["beta"] / P                              # d loss / d seq of the chosen summary
        cs = torch.cat([dh, -dh])
        if c["average"]:
            cs = cs / cnt
        coef = torch.where(keep, cs[:, None], torch.zeros_like(lp))
        return {"loss": loss, "margins": h, "dlogits": _plain_dlogits(p, lab, coef, s["logits"].dtype)}
    w = torch.where(keep, (1.0 / keep.sum().clamp(min=1).float()) if c["reduction"] == "token" else (1.0 / (cnt * c["N"]))[:, None], 0.0)
    ratio = torch.where(keep, torch.exp(lp - s["old"]), torch.ones_like(lp))
    a = s["adv"][:, None]
    l1, l2 = -a * ratio, -a * ratio.clamp(1 - c["low"], 1 + c["high"])
    pg, dlp = torch.maximum(l1, l2), torch.where(l1 >= l2, l1, torch.zeros_like(l1))
    kl = torch.zeros_like(lp)
    if s["ref"] is not None:
        d = torch.where(keep, s["ref"] - lp, torch.zeros_like(lp))
        kl = torch.exp(d) - d - 1.0
        dlp = dlp + c["kl"] * (1.0 - torch.exp(d))
    return {"loss": (w * (pg + c["kl"] * kl)).sum(), "kl": (w * kl).sum(), "clipped": (w * (l1 < l2)).sum(), "token": lp,
            "dlogits": _plain_dlogits(p, lab, w * dlp, s["logits"].dtype)}


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


# ---------------------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    d = _inputs(c, seed)
    f8 = torch.float64
    if c["kind"] == "i8":
        top_x, top_w = d["x"].to(f8).abs().max(1).values, d["w"].to(f8).abs().max(1).values
        sw = (top_w.float() / 127.0).to(f8)                                        # scales are held in 32 bits
        wv = torch.round(d["w"].to(f8) * 127.0 / top_w[:, None]).t().contiguous()
        parts = []
        for lo in range(0, c["M"], 4096):
            top = top_x[lo:lo + 4096]
            q = torch.nan_to_num(torch.round(d["x"][lo:lo + 4096].to(f8) * 127.0 / top[:, None]))
            y = torch.mm(q, wv) * (top.float() / 127.0).to(f8)[:, None] * sw
            y = y if d["bias"] is None else y + d["bias"].to(f8)
            parts.append(y * (1.0 + torch.special.erf(y / math.sqrt(2.0))) / 2.0 if c["gelu"] else y)
        return torch.cat(parts)
    if c["kind"] == "embed":
        ids = d["ids"].flatten()
        grad = torch.zeros(c["V"], c["D"], dtype=f8, device=ids.device)
        real = ids != 1
        grad.index_put_((ids[real],), d["dy"].reshape(-1, c["D"])[real].to(f8) * c["scale"], accumulate=True)
        return {"y": d["table"].to(f8)[ids].reshape(c["N"], c["T"], c["D"]) * c["scale"], "dtable": grad}
    N, T = c["N"], c["T"]
    lens = _lengths(c)
    logp = torch.zeros(N, T, dtype=f8, device="cuda")
    for n in range(N):
        if lens[n]:
            x = torch.log_softmax(d["logits"][n, :lens[n]].to(f8), -1)
            logp[n, :lens[n]] = x[torch.arange(lens[n], device="cuda"), d["labels"][n, :lens[n]]]
    cnt = torch.tensor([float(max(1, v)) for v in lens], dtype=f8, device="cuda")
    mask = torch.arange(T, device="cuda")[None, :] < torch.tensor(lens, device="cuda")[:, None]
    seq = logp.sum(1) / (cnt if c.get("average") else 1.0)
    if c["kind"] == "score":
        return {"sequence": seq, "token": logp}
    if c["kind"] == "pref":
        P, eps = N // 2, c["smoothing"]
        leaf = seq.clone().requires_grad_(True)
        gap = leaf - d["ref"].to(f8)
        h = c["beta"] * (gap[:P] - gap[P:])
        loss = -((1 - eps) * torch.nn.functional.logsigmoid(h) + eps * torch.nn.functional.logsigmoid(-h)).mean()
        loss.backward()
        coef = (leaf.grad / (cnt if c["average"] else 1.0))[:, None] * mask
        out = {"loss": loss.detach(), "margins": h.detach()}
    else:
        weight = mask / (max(1, sum(lens)) if c["reduction"] == "token" else cnt[:, None] * N)
        leaf = logp.clone().requires_grad_(True)
        ratio = (leaf - d["old"].to(f8)).exp()
        a = d["adv"].to(f8)[:, None]
        bounded = torch.minimum(torch.maximum(ratio, torch.full_like(ratio, 1 - c["low"])), torch.full_like(ratio, 1 + c["high"]))
        gain = torch.minimum(a * ratio, a * bounded)
        kl = torch.zeros_like(logp)
        if d["ref"] is not None:
            gap = d["ref"].to(f8) - leaf
            kl = gap.exp() - 1.0 - gap
        loss = (weight * (c["kl"] * kl - gain)).sum()
        loss.backward()
        coef = leaf.grad * mask
        out = {"loss": loss.detach(), "kl": (weight * kl).sum().detach(), "clipped": (weight * (a * bounded < a * ratio)).sum().detach(), "token": logp}
    dl = torch.zeros(N, T, c["V"], dtype=f8, device="cuda")
    for n in range(N):
        for_n = -torch.softmax(d["logits"][n, :lens[n]].to(f8), -1)
        for_n[torch.arange(lens[n], device="cuda"), d["labels"][n, :lens[n]]] += 1.0
        dl[n, :lens[n]] = for_n * coef[n, :lens[n], None]
    out["dlogits"] = dl
    return out
