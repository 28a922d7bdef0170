"""The operators of a packed training step around the loss, as they are measured:
cases over their real range, the operators in plain torch, the calls of this
package, and their values in 64 bits.

Three operators:

  attention   causal attention of the packed row the loss is taken over: every
              token sees the tokens of its own document up to itself, the
              document's prompt whole where it has a prefix, at most `window`
              tokens back; scores capped by a tanh where the model caps them;
              several query heads share a key and value head.  "train" returns
              the gradients too, "eval" the output alone.
  norm        what stands between two blocks of a decoder: the block's output,
              normalised where the model norms after the block too, gated and
              scaled, is added to the residual, and the sum normalised for the
              next block; forward and backward.
  clip        the global norm of all gradients of a step, and their scaling in
              place to a largest norm.

The documents of a packed row have lognormal lengths, as the loss's cases have.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}

# Flops of the largest attention case, elements of the largest norm and of the
# largest set of gradients: no drawn case costs more.
MOST_FLOPS = 7.0e12
MOST_ROW_ELEMENTS = 65536 * 4096
MOST_GRADIENTS = 1_500_000_000


def _attention(direction, dtype, T, docs, heads, kv_heads, D, softcap=0.0, window=0, prefix=0.0,
               pad=0, spread=0.8):
    return {"kind": "attention", "direction": direction, "dtype": dtype, "T": T, "docs": docs,
            "heads": heads, "kv_heads": kv_heads, "D": D, "softcap": softcap, "window": window,
            "prefix": prefix, "pad": pad, "spread": spread}


def _norm(dtype, T, H, post=False, gate="none", block_scale=1.0, residual_scale=1.0, offset=0.0):
    return {"kind": "norm", "dtype": dtype, "T": T, "H": H, "post": post, "gate": gate,
            "block_scale": block_scale, "residual_scale": residual_scale, "offset": offset}


def _clip(layers, H, I, kv, V, clips, accumulator):
    return {"kind": "clip", "layers": layers, "H": H, "I": I, "kv": kv, "V": V, "clips": clips,
            "accumulator": accumulator}


def listed():
    return [
        # a toy model or a unit test's step: launches and host work are all of it
        {"name": "attention_tiny", **_attention("train", "bf16", 192, 4, 4, 2, 64)},
        # the ordinary minibatch: a few thousand packed tokens through an 8B model's heads
        {"name": "attention_4k", **_attention("train", "bf16", 4096, 12, 32, 8, 128)},
        # a large packed minibatch of a small model, which has few key heads
        {"name": "attention_32k_packed", **_attention("train", "bf16", 32768, 64, 12, 2, 128)},
        # one long document through an 8B model's heads, scores capped
        {"name": "attention_16k_softcap",
         **_attention("train", "bf16", 16384, 1, 32, 8, 128, softcap=50.0)},
        # evaluation of one long document
        {"name": "attention_32k_eval", **_attention("eval", "bf16", 32768, 1, 32, 8, 128)},
        # ragged everything: odd lengths, prompts seen whole, a local layer's window,
        # capped scores, rows behind the last document
        {"name": "attention_ragged",
         **_attention("train", "bf16", 3001, 7, 14, 2, 64, softcap=30.0, window=300, prefix=0.3,
                      pad=57)},
        # a model kept in fp32
        {"name": "attention_fp32", **_attention("train", "fp32", 2048, 8, 14, 2, 64)},
        # a toy model's step
        {"name": "norm_tiny", **_norm("bf16", 192, 128)},
        # the headline's packed row: residual and pre-norm alone
        {"name": "norm_64k", **_norm("bf16", 65536, 4096)},
        # norms before and after the block, a gate for each channel, both scales
        {"name": "norm_sandwich", **_norm("bf16", 16384, 3584, post=True, gate="channel",
                                          block_scale=0.22, residual_scale=0.9, offset=1.0)},
        # all gradients of a toy model
        {"name": "clip_tiny", **_clip(2, 128, 352, 64, 1000, True, False)},
        # all gradients of a 1.5B model, its head's in an fp32 accumulator
        {"name": "clip_1b", **_clip(28, 1536, 8960, 256, 151936, True, True)},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["attention"] * 3 + ["norm"] * 2 + ["clip"])
    if kind == "norm":
        H = _log_int(rng, 64, 8192)
        r = rng.random()
        H = H // 64 * 64 if r < 0.7 else H // 8 * 8 if r < 0.9 else H
        T = _log_int(rng, 1, min(65536, MOST_ROW_ELEMENTS // H))
        post = rng.random() < 0.5
        return _norm("fp32" if rng.random() < 0.25 else "bf16", T, H, post,
                     rng.choice(["none", "none", "channel", "token"]),
                     rng.choice([1.0, round(rng.uniform(0.1, 1.0), 2)]),
                     rng.choice([1.0, round(rng.uniform(0.5, 1.5), 2)]),
                     rng.choice([0.0, 1.0]))
    if kind == "clip":
        H = _log_int(rng, 64, 4096) // 8 * 8
        layers = _log_int(rng, 1, 32)
        V = _log_int(rng, 1000, 152064)
        I = int(H * rng.uniform(2.0, 4.0))
        while layers > 1 and layers * H * (3 * I + 3 * H) + 3 * V * H > MOST_GRADIENTS:
            layers -= 1
        V = max(1000, min(V, (MOST_GRADIENTS - layers * H * (3 * I + 3 * H)) // (3 * H)))
        return _clip(layers, H, I, max(8, H // rng.choice([1, 4, 8])), V, rng.random() < 0.6,
                     rng.random() < 0.4)
    dtype = "fp32" if rng.random() < 0.2 else "bf16"
    D = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 7])
    direction = rng.choice(["train", "train", "eval"])
    T = _log_int(rng, 1, 32768)
    docs = _log_int(rng, 1, min(256, max(1, T // 8)))
    # one document of the whole length is the costliest: fp32 runs an order of
    # magnitude slower, so less of it is drawn
    per_pair = (14.0 if direction == "train" else 4.0) * D * heads
    most = MOST_FLOPS / (16 if dtype == "fp32" else 1)
    T = min(T, int(math.sqrt(2.0 * most / per_pair)))
    docs = min(docs, T)
    pad = rng.choice([0, 0, rng.randrange(0, T - docs + 1)]) if T > docs else 0
    return _attention(direction, dtype, T, docs, heads, kv, D,
                      rng.choice([0.0, 0.0, 30.0, 50.0]),
                      rng.choice([0, 0, _log_int(rng, 1, 4096)]),
                      rng.choice([0.0, 0.0, round(rng.uniform(0.1, 0.9), 2)]),
                      min(pad, T // 4), round(rng.uniform(0.3, 1.2), 2))


def _generator(seed, k):
    return torch.Generator(device="cuda").manual_seed(seed * 1009 + k)


def _normal(shape, dtype, seed, k, std=1.0):
    x = torch.randn(shape, generator=_generator(seed, k), device="cuda", dtype=torch.float32)
    return x.mul_(std).to(DTYPES[dtype])


def _lengths(case):
    """The documents' lengths: the same for every seed, which gives their order."""
    n, S = case["T"] - case["pad"], case["docs"]
    g = torch.Generator().manual_seed(17)
    raw = torch.exp(case["spread"] * torch.randn(S, generator=g, dtype=torch.float64))
    lengths = torch.clamp((raw * (n - S) / raw.sum()).floor().long() + 1, min=1)
    lengths[int(lengths.argmax())] += n - int(lengths.sum())
    return lengths


def _documents(case, lengths):
    """[start, end, end of the prefix) of each document, on the host."""
    at, spans = 0, []
    for n in lengths.tolist():
        spans.append((at, at + n, at + int(case["prefix"] * n)))
        at += n
    return spans


def _row_ranges(case, spans, device):
    """The range [lo, hi) of keys each row of the packed documents sees."""
    T, w = case["T"], case["window"] or case["T"]
    start, end, seen = (torch.tensor([s[k] for s in spans], device=device) for k in range(3))
    counts = end - start
    rows = torch.arange(int(spans[-1][1]), device=device)
    first, prompt = (torch.repeat_interleave(x, counts) for x in (start, seen))
    return torch.maximum(first, rows - w + 1), torch.maximum(rows + 1, prompt)


def _prepare_attention(case, seed):
    order = torch.randperm(case["docs"], generator=torch.Generator().manual_seed(seed))
    lengths = _lengths(case)[order]
    spans = _documents(case, lengths)
    T, D, dt = case["T"], case["D"], case["dtype"]
    s = {"case": case, "spans": spans}
    s["cu_seqlens"] = torch.tensor([0] + [e for _, e, _ in spans], dtype=torch.int32, device="cuda")
    s["prefix_lens"] = None
    if case["prefix"]:
        s["prefix_lens"] = torch.tensor([p - a for a, _, p in spans], dtype=torch.int32,
                                        device="cuda")
    train = case["direction"] == "train"
    # queries wider than keys: scores of standard deviation 2, as trained heads have
    s["q"] = _normal((T, case["heads"], D), dt, seed, 1, 2.0).requires_grad_(train)
    s["k"] = _normal((T, case["kv_heads"], D), dt, seed, 2).requires_grad_(train)
    s["v"] = _normal((T, case["kv_heads"], D), dt, seed, 3).requires_grad_(train)
    if train:
        s["dout"] = _normal((T, case["heads"], D), dt, seed, 4)
    return s


def _prepare_norm(case, seed):
    T, H, dt = case["T"], case["H"], case["dtype"]
    s = {"case": case}
    s["x"] = _normal((T, H), dt, seed, 1, 1.5).requires_grad_(True)
    s["residual"] = _normal((T, H), dt, seed, 2, 3.0).requires_grad_(True)
    s["weight"] = (_normal((H,), "fp32", seed, 3, 0.2) + (1.0 - case["offset"])) \
        .to(DTYPES[dt]).requires_grad_(True)
    s["post_weight"] = s["gate"] = None
    if case["post"]:
        s["post_weight"] = (_normal((H,), "fp32", seed, 4, 0.2) + (1.0 - case["offset"])) \
            .to(DTYPES[dt]).requires_grad_(True)
    if case["gate"] != "none":
        shape = (H,) if case["gate"] == "channel" else (T, 1)
        s["gate"] = (_normal(shape, "fp32", seed, 5, 0.5) + 1.0).to(DTYPES[dt]).requires_grad_(True)
    s["dnormed"] = _normal((T, H), dt, seed, 6)
    s["dresidual"] = _normal((T, H), dt, seed, 7)
    return s


def _shapes(case):
    """(bf16 gradients, fp32 gradients) of a decoder's parameters."""
    H, I, kv, V = (case[k] for k in ("H", "I", "kv", "V"))
    layer = [(H, H), (H,), (kv, H), (kv,), (kv, H), (kv,), (H, H), (I, H), (I, H), (H, I), (H,),
             (H,)]
    narrow = [(V, H)] + layer * case["layers"] + [(H,)]
    return (narrow, [(V, H)]) if case["accumulator"] else (narrow + [(V, H)], [])


def _numbers(shapes):
    return [math.prod(x) for x in shapes]


def _prepare_clip(case, seed):
    s = {"case": case, "flat": [], "gradients": []}
    total = 0
    for k, (shapes, dt) in enumerate(zip(_shapes(case), ("bf16", "fp32"))):
        if not shapes:
            continue
        # each gradient from a 16-byte boundary on, as an allocator places them
        sizes = [-(-n // 8) * 8 for n in _numbers(shapes)]
        flat = _normal((sum(sizes),), dt, seed, k, 1e-3)
        at = 0
        for shape, n, size in zip(shapes, _numbers(shapes), sizes):
            flat[at + n:at + size] = 0
            s["gradients"].append(flat[at:at + n].view(shape))
            at += size
        s["flat"].append(flat)
        total += sum(_numbers(shapes))
    s["max_norm"] = 1e-3 * math.sqrt(total) * (0.37 if case["clips"] else 2.0)
    return s


def prepare(case, seed):
    return {"attention": _prepare_attention, "norm": _prepare_norm,
            "clip": _prepare_clip}[case["kind"]](case, seed)


def _row_blocks(spans, heads):
    """Rows of one document at a time, few enough for their scores in 1 GiB."""
    blocks = []
    for a, e, _ in spans:
        step = max(1, (1 << 28) // (heads * (e - a)))
        blocks += [(a, e, r, min(e, r + step)) for r in range(a, e, step)]
    return blocks


def _plain_attention(s):
    case = s["case"]
    T, Hq, Hk, D, cap = (case[k] for k in ("T", "heads", "kv_heads", "D", "softcap"))
    G, dt, train = Hq // Hk, s["q"].dtype, case["direction"] == "train"
    lo, hi = _row_ranges(case, s["spans"], "cuda")

    def heads_first(x):  # [T, Hq, D] -> [Hk, G, T, D]
        return x.detach().float().view(T, Hk, -1, D).permute(1, 2, 0, 3)

    q, k, v = heads_first(s["q"]) * D ** -0.5, heads_first(s["k"])[:, 0], heads_first(s["v"])[:, 0]
    out, dq = torch.zeros((2, Hk, G, T, D), device="cuda").unbind(0)
    dk, dv = torch.zeros((2, Hk, T, D), device="cuda").unbind(0)
    dout = heads_first(s["dout"]) if train else None
    for a, e, r0, r1 in _row_blocks(s["spans"], Hq):
        kb, vb = k[:, a:e], v[:, a:e]
        qb = q[:, :, r0:r1].reshape(Hk, -1, D)
        z = qb @ kb.transpose(1, 2)
        if cap:
            t = torch.tanh(z / cap)
            z = cap * t
        key = torch.arange(a, e, device="cuda")
        hidden = (key < lo[r0:r1, None]) | (key >= hi[r0:r1, None])
        z = z.view(Hk, G, r1 - r0, e - a).masked_fill(hidden, -math.inf).view(Hk, -1, e - a)
        p = torch.exp(z - z.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        out[:, :, r0:r1] = (p @ vb).view(Hk, G, r1 - r0, D)
        if train:
            db = dout[:, :, r0:r1].reshape(Hk, -1, D)
            dv[:, a:e] += p.transpose(1, 2) @ db
            dp = db @ vb.transpose(1, 2)
            dz = p * (dp - (p * dp).sum(-1, keepdim=True))
            if cap:
                dz = dz * (1 - t * t)
            dq[:, :, r0:r1] = (dz @ kb).view(Hk, G, r1 - r0, D) * D ** -0.5
            dk[:, a:e] += dz.transpose(1, 2) @ qb

    def tokens_first(x):
        return x.permute(2, 0, 1, 3).reshape(T, Hq, D).to(dt)

    if not train:
        return {"out": tokens_first(out)}
    return {"out": tokens_first(out), "dq": tokens_first(dq),
            "dk": dk.transpose(0, 1).contiguous().to(dt),
            "dv": dv.transpose(0, 1).contiguous().to(dt)}


EPS = 1e-6


def _plain_norm(s):
    case = s["case"]
    dt = s["x"].dtype
    x, r, w, dn, dr = (s[k].detach().float() for k in ("x", "residual", "weight", "dnormed",
                                                       "dresidual"))
    w = w + case["offset"]
    g = 1.0 if s["gate"] is None else s["gate"].detach().float()
    u = x
    if case["post"]:
        pw = s["post_weight"].detach().float() + case["offset"]
        ix = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        xn = x * ix
        u = xn * pw
    h = case["residual_scale"] * r + case["block_scale"] * (g * u)
    ih = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    hn = h * ih
    out = {"normed": (hn * w).to(dt), "residual": h.to(dt)}
    out["dweight"] = (dn * hn).sum(0).to(dt)
    dhn = dn * w
    dh = dr + ih * (dhn - hn * (dhn * hn).mean(-1, keepdim=True))
    out["dresidual"] = (case["residual_scale"] * dh).to(dt)
    du = case["block_scale"] * g * dh
    if s["gate"] is not None:
        dg = case["block_scale"] * dh * u
        out["dgate"] = (dg.sum(0) if case["gate"] == "channel" else dg.sum(1, keepdim=True)).to(dt)
    if case["post"]:
        out["dpost_weight"] = (du * xn).sum(0).to(dt)
        dxn = du * pw
        du = ix * (dxn - xn * (dxn * xn).mean(-1, keepdim=True))
    out["dx"] = du.to(dt)
    return out


def _clip_bound(s):
    """The largest norm of this pass: it falls a little from pass to pass, so
    that each pass over gradients scaled before scales them again."""
    bound = s["max_norm"]
    if s["case"]["clips"]:
        s["max_norm"] = bound * 0.999
    return bound


def _plain_clip(s):
    bound = _clip_bound(s)
    squares = [g.double().square().sum() for g in s["gradients"]]
    norm = torch.stack(squares).sum().sqrt()
    scale = torch.clamp(bound / (norm + 1e-6), max=1.0).float()
    for g in s["gradients"]:
        g.copy_(g.float() * scale)
    return {"norm": norm.float(), "gradients": s["flat"]}


def _run_own(s):
    from mini_trainer_amd import (clip_gradients_, packed_attention, packed_attention_plan,
                                  residual_rms_norm)

    case = s["case"]
    if case["kind"] == "clip":
        return {"norm": clip_gradients_(s["gradients"], _clip_bound(s)), "gradients": s["flat"]}
    if case["kind"] == "norm":
        normed, residual = residual_rms_norm(
            s["x"], s["residual"], s["weight"], eps=EPS, post_weight=s["post_weight"],
            gate=s["gate"], block_scale=case["block_scale"],
            residual_scale=case["residual_scale"], weight_offset=case["offset"])
        names = [n for n in ("x", "residual", "weight", "post_weight", "gate") if s[n] is not None]
        grads = torch.autograd.grad([normed, residual], [s[n] for n in names],
                                    [s["dnormed"], s["dresidual"]])
        return {"normed": normed, "residual": residual,
                **{"d" + n: d for n, d in zip(names, grads)}}
    plan = packed_attention_plan(s["cu_seqlens"], case["T"], window=case["window"] or None,
                                 prefix_lens=s["prefix_lens"], validate=False)
    out = packed_attention(s["q"], s["k"], s["v"], plan, softcap=case["softcap"] or None)
    if case["direction"] == "eval":
        return {"out": out}
    grads = torch.autograd.grad(out, [s["q"], s["k"], s["v"]], s["dout"])
    return {"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]}


def run(state):
    if own:
        return _run_own(state)
    return {"attention": _plain_attention, "norm": _plain_norm,
            "clip": _plain_clip}[state["case"]["kind"]](state)


def _pairs(case):
    """(query, key) pairs that see each other; the same in any order of the documents."""
    w = case["window"] or case["T"]
    total = 0
    for n in _lengths(case).tolist():
        p = int(case["prefix"] * n)
        i = torch.arange(n, dtype=torch.int64)
        total += int((torch.clamp(i + 1, min=p) - torch.clamp(i - w + 1, min=0)).sum())
    return total


def work(case):
    if case["kind"] == "clip":
        narrow, wide = (sum(_numbers(x)) for x in _shapes(case))
        n, size = narrow + wide, 2 * narrow + 4 * wide
        return {"bytes": size * (2 if case["clips"] else 1),
                "flops": n * (3 if case["clips"] else 2)}
    es = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "norm":
        n = case["T"] * case["H"]
        # x, residual, two upstream gradients in; two outputs, two gradients out
        return {"bytes": 8 * n * es, "flops": n * (40 if case["post"] else 24)}
    train = case["direction"] == "train"
    q, kv = case["T"] * case["heads"] * case["D"], case["T"] * case["kv_heads"] * case["D"]
    return {"bytes": es * (4 * q + 4 * kv if train else 2 * q + 2 * kv),
            "flops": (14 if train else 4) * case["D"] * case["heads"] * _pairs(case)}


def _exact_attention(case, s):
    Hk, G, D = case["kv_heads"], case["heads"] // case["kv_heads"], case["D"]
    window, train = case["window"], case["direction"] == "train"
    grown = {n: s[n].detach().double().requires_grad_(train) for n in ("q", "k", "v")}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    grads = {n: torch.zeros_like(x, requires_grad=False) for n, x in grown.items()}
    for a, e, p in s["spans"]:
        i = torch.arange(a, e, device="cuda")[:, None]
        j = torch.arange(a, e, device="cuda")[None, :]
        sees = (j <= i) | (j < p)
        if window:
            sees &= i - j < window
        for h in range(Hk):
            part = [grown["q"][a:e, h * G:(h + 1) * G].detach().requires_grad_(train),
                    grown["k"][a:e, h].detach().requires_grad_(train),
                    grown["v"][a:e, h].detach().requires_grad_(train)]
            for g in range(G):
                score = part[0][:, g] @ part[1].T / math.sqrt(D)
                if case["softcap"]:
                    score = case["softcap"] * torch.tanh(score / case["softcap"])
                y = torch.softmax(torch.where(sees, score, -math.inf), -1) @ part[2]
                out[a:e, h * G + g] = y.detach()
                if train:
                    got = torch.autograd.grad(y, part, s["dout"][a:e, h * G + g].double())
                    grads["q"][a:e, h * G:(h + 1) * G] += got[0]
                    grads["k"][a:e, h] += got[1]
                    grads["v"][a:e, h] += got[2]
                del score, y
    if not train:
        return {"out": out}
    return {"out": out, "dq": grads["q"], "dk": grads["k"], "dv": grads["v"]}


def _exact_norm(case, s):
    names = [n for n in ("x", "residual", "weight", "post_weight", "gate") if s[n] is not None]
    at = {n: s[n].detach().double().requires_grad_(True) for n in names}

    def rms(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * (case["offset"] + w)

    block = rms(at["x"], at["post_weight"]) if case["post"] else at["x"]
    if "gate" in at:
        block = at["gate"] * block
    total = case["residual_scale"] * at["residual"] + case["block_scale"] * block
    normed = rms(total, at["weight"])
    grads = torch.autograd.grad([normed, total], [at[n] for n in names],
                                [s["dnormed"].double(), s["dresidual"].double()])
    return {"normed": normed.detach(), "residual": total.detach(),
            **{"d" + n: g for n, g in zip(names, grads)}}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        if case["docs"] * case["heads"] > 10000:
            return None
        return _exact_attention(case, s)
    if case["kind"] == "norm":
        return _exact_norm(case, s)
    flat = [f.double() for f in s["flat"]]
    norm = math.sqrt(sum(float(torch.dot(f, f)) for f in flat))
    return {"norm": torch.tensor(norm, dtype=torch.float64),
            "gradients": [f * min(1.0, s["max_norm"] / (norm + 1e-6)) for f in flat]}
