"""Operators at the two ends of a packed training step and in its layers, as they are
measured: cases over their real range, the operators in plain torch, the calls of
this package, and their values in 64 bits.

Three operators:

  embedding      the rows of the token embedding that a packed row of token ids asks
                 for, times a scale where the model scales them, and the weight's
                 gradient: the sum of the upstream gradient's rows for each token,
                 returned whole or added to the fp32 accumulator that the loss's head
                 gradient goes to as well.
  layer_norm     the layer norm of the decoders that have no RMS norm: of a tensor, or
                 of a block's output added to the residual, which is then returned
                 too; forward and backward, the weight's and the bias's gradients
                 among it.
  orthogonalize  the orthogonalised update of weight matrices: Newton-Schulz steps
                 on the momentum divided by its norm, for one matrix or a stack of
                 them.

Token ids follow Zipf's law, as a tokenizer's do: low ids are the frequent ones.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NORM_EPS = 1e-5
UPDATE_EPS = 1e-7

# Elements of the largest embedding (rows looked up and rows of the weight), of the
# largest norm and flops of the largest update: no drawn case costs more.
MOST_EMBEDDED = (65536 + 128256) * 4096
MOST_NORMED = 32768 * 4096
MOST_FLOPS = 5 * (3 * 4096 ** 2 * 14336 + 4096 ** 3)


def _embedding(dtype, T, V, H, scale=1.0, gradient="whole", padding=0, ids="int64"):
    return {"kind": "embedding", "dtype": dtype, "T": T, "V": V, "H": H, "scale": scale,
            "gradient": gradient, "padding": padding, "ids": ids}


def _layer_norm(dtype, T, H, residual=True, bias=True, direction="train", block_scale=1.0,
                residual_scale=1.0):
    return {"kind": "layer_norm", "dtype": dtype, "T": T, "H": H, "residual": residual,
            "bias": bias, "direction": direction, "block_scale": block_scale,
            "residual_scale": residual_scale}


def _orthogonalize(dtype, batch, m, n):
    return {"kind": "orthogonalize", "dtype": dtype, "batch": batch, "m": m, "n": n}


def listed():
    return [
        # a toy model or a unit test's step: launches and host work are all of it
        {"name": "embedding_tiny", **_embedding("bf16", 192, 1000, 128)},
        # the headline's packed row through an 8B model's embedding, its gradient whole
        {"name": "embedding_64k", **_embedding("bf16", 65536, 128256, 4096)},
        # a 1.5B model with tied embeddings: the gradient joins the head's in fp32
        {"name": "embedding_tied",
         **_embedding("bf16", 16384, 151936, 1536, gradient="accumulate")},
        # a model in fp32 that scales its embeddings, odd sizes, rows of padding
        {"name": "embedding_fp32_odd",
         **_embedding("fp32", 3001, 50257, 1030, scale=32.094, padding=411, ids="int32")},
        # a toy model's step
        {"name": "norm_tiny", **_layer_norm("bf16", 192, 128)},
        # half the headline's packed row: residual and norm, forward and backward
        {"name": "norm_32k", **_layer_norm("bf16", 32768, 4096)},
        # a model kept in fp32, a width of no whole vectors, a norm without a bias at
        # the decoder's end
        {"name": "norm_fp32_odd", **_layer_norm("fp32", 2999, 1601, residual=False, bias=False)},
        # one matrix of a toy model
        {"name": "update_tiny", **_orthogonalize("bf16", 1, 128, 352)},
        # the key projections of all layers of a 1.5B model at once
        {"name": "update_keys", **_orthogonalize("bf16", 28, 256, 1536)},
        # an 8B model's attention projection
        {"name": "update_square", **_orthogonalize("bf16", 1, 4096, 4096)},
        # an 8B model's MLP weight, taller than wide
        {"name": "update_tall", **_orthogonalize("bf16", 1, 14336, 4096)},
        # matrices of odd sizes in fp32
        {"name": "update_fp32_odd", **_orthogonalize("fp32", 3, 1001, 1537)},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _width(rng, lo, hi):
    """A width: most often whole vectors, now and then an odd one."""
    H, r = _log_int(rng, lo, hi), rng.random()
    return (H // 64 * 64 if r < 0.6 else H // 8 * 8 if r < 0.8 else H) or H


def _update_flops(m, n):
    """Flops of an update: three products a step, of which two are symmetric."""
    r, c = min(m, n), max(m, n)
    return STEPS * (3 * r * r * c + r ** 3)


def draw(rng):
    kind = rng.choice(["embedding", "layer_norm", "orthogonalize"])
    dtype = "fp32" if rng.random() < 0.3 else "bf16"
    if kind == "embedding":
        H = _width(rng, 16, 8192)
        most = MOST_EMBEDDED // H // (2 if dtype == "fp32" else 1)
        V = _log_int(rng, 100, min(262144, most * 2 // 3))
        T = _log_int(rng, 1, min(131072, most - V))
        return _embedding(dtype, T, V, H, rng.choice([1.0, 1.0, round(math.sqrt(H), 3)]),
                          rng.choice(["whole", "accumulate"]),
                          rng.choice([0, 0, rng.randrange(0, T // 3 + 1)]),
                          rng.choice(["int64", "int64", "int32"]))
    if kind == "layer_norm":
        H = _width(rng, 64, 8192)
        T = _log_int(rng, 1, min(65536, MOST_NORMED // H // (2 if dtype == "fp32" else 1)))
        residual = rng.random() < 0.7
        scales = [rng.choice([1.0, round(rng.uniform(0.1, 1.5), 2)]) if residual else 1.0
                  for _ in range(2)]
        return _layer_norm(dtype, T, H, residual, rng.random() < 0.7,
                           rng.choice(["train", "train", "eval"]), *scales)
    m, n = _width(rng, 1, 8192), _width(rng, 1, 16384)
    if rng.random() < 0.3:
        n = m
    # fp32 takes three products for each of bf16's
    most = MOST_FLOPS // (4 if dtype == "fp32" else 1)
    while _update_flops(m, n) > most:
        m, n = max(1, m * 4 // 5), max(1, n * 4 // 5)
    batch = _log_int(rng, 1, min(64, max(1, most // _update_flops(m, n)),
                                 max(1, 200_000_000 // (m * n))))
    return _orthogonalize(dtype, batch, m, n)


def _generator(seed, k):
    return torch.Generator(device="cuda").manual_seed(seed * 1009 + k)


def _normal(shape, dtype, seed, k, std=1.0):
    x = torch.randn(shape, generator=_generator(seed, k), device="cuda", dtype=torch.float32)
    return x.mul_(std).to(DTYPES[dtype])


def _zipf(V):
    """Probabilities of the ids, the frequent ones first."""
    p = 1.0 / (torch.arange(V, dtype=torch.float64) + 2.7)
    return p / p.sum()


def _padding_id(case):
    return case["V"] - 1 if case["padding"] else None


def _prepare_embedding(case, seed):
    T, V, H, dt = case["T"], case["V"], case["H"], case["dtype"]
    s = {"case": case}
    cumulative = torch.cumsum(_zipf(V), 0).cuda()
    at = torch.rand(T, generator=_generator(seed, 1), device="cuda", dtype=torch.float64)
    ids = torch.searchsorted(cumulative, at, right=True).clamp_(max=V - 1)
    if case["padding"]:
        ids[T - case["padding"]:] = V - 1
    s["ids"] = ids.to(getattr(torch, case["ids"]))
    s["weight"] = _normal((V, H), dt, seed, 2, 0.02).requires_grad_(True)
    s["dout"] = _normal((T, H), dt, seed, 3, 1e-2)
    s["accumulator"] = None
    if case["gradient"] == "accumulate":
        s["accumulator"] = _normal((V, H), "fp32", seed, 4, 1e-2)
    return s


def _prepare_layer_norm(case, seed):
    T, H, dt = case["T"], case["H"], case["dtype"]
    train = case["direction"] == "train"
    s = {"case": case, "residual": None, "bias": None}
    s["x"] = _normal((T, H), dt, seed, 1, 1.5)
    if case["residual"]:
        # channels of a residual stream have means of their own
        mean = _normal((H,), "fp32", seed, 2, 1.0)
        s["residual"] = (_normal((T, H), "fp32", seed, 3, 2.0) + mean + 0.5).to(DTYPES[dt])
    s["weight"] = (_normal((H,), "fp32", seed, 4, 0.2) + 1.0).to(DTYPES[dt])
    if case["bias"]:
        s["bias"] = _normal((H,), dt, seed, 5, 0.3)
    if train:
        for n in ("x", "residual", "weight", "bias"):
            if s[n] is not None:
                s[n].requires_grad_(True)
        s["dnormed"] = _normal((T, H), dt, seed, 6)
        s["dresidual"] = _normal((T, H), dt, seed, 7) if case["residual"] else None
    return s


def _prepare_orthogonalize(case, seed):
    """Momenta: a few strong directions, as sums of outer products have them, over
    noise."""
    batch, m, n = case["batch"], case["m"], case["n"]
    k = max(1, min(m, n) // 8)
    rows = _normal((batch, m, k), "fp32", seed, 1)
    strength = torch.exp(_normal((batch, 1, k), "fp32", seed, 2))
    columns = _normal((batch, k, n), "fp32", seed, 3)
    update = torch.bmm(rows * strength, columns).div_(math.sqrt(k))
    update += _normal((batch, m, n), "fp32", seed, 4)
    update = update.mul_(1e-3).to(DTYPES[case["dtype"]])
    return {"case": case, "update": update if batch > 1 else update[0]}


def prepare(case, seed):
    return {"embedding": _prepare_embedding, "layer_norm": _prepare_layer_norm,
            "orthogonalize": _prepare_orthogonalize}[case["kind"]](case, seed)


def _plain_embedding(s):
    case = s["case"]
    dt, ids, scale = s["weight"].dtype, s["ids"].long(), case["scale"]
    out = (s["weight"].detach()[ids].float() * scale).to(dt)
    d = s["dout"].float() * scale
    if case["padding"]:
        d = d * (ids != _padding_id(case))[:, None]
    if s["accumulator"] is not None:
        s["accumulator"].index_add_(0, ids, d)
        return {"out": out, "accumulator": s["accumulator"]}
    dweight = torch.zeros((case["V"], case["H"]), device="cuda").index_add_(0, ids, d)
    return {"out": out, "dweight": dweight.to(dt)}


def _plain_layer_norm(s):
    case, dt = s["case"], s["x"].dtype
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    h = x
    if case["residual"]:
        h = case["residual_scale"] * s["residual"].detach().float() + case["block_scale"] * x
    centred = h - h.mean(-1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(-1, keepdim=True) + NORM_EPS)
    hn = centred * rstd
    y = hn * w
    if case["bias"]:
        y = y + s["bias"].detach().float()
    out = {"normed": y.to(dt)}
    if case["residual"]:
        out["residual"] = h.to(dt)
    if case["direction"] == "eval":
        return out
    dy = s["dnormed"].float()
    out["dweight"] = (dy * hn).sum(0).to(dt)
    if case["bias"]:
        out["dbias"] = dy.sum(0).to(dt)
    d = dy * w
    dh = rstd * (d - d.mean(-1, keepdim=True) - hn * (d * hn).mean(-1, keepdim=True))
    if case["residual"]:
        dh = dh + s["dresidual"].float()
        out["dresidual"] = (case["residual_scale"] * dh).to(dt)
        dh = case["block_scale"] * dh
    out["dx"] = dh.to(dt)
    return out


def _plain_orthogonalize(s):
    a, b, c = COEFFICIENTS
    x = s["update"].float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT.contiguous()
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = x * (1.0 / (norm + UPDATE_EPS)).float()
    for _ in range(STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return {"out": (x.mT if tall else x).to(s["update"].dtype).contiguous()}


def _run_own(s):
    from mini_trainer_amd import layer_norm, orthogonalize, residual_layer_norm, token_embedding

    case = s["case"]
    if case["kind"] == "orthogonalize":
        return {"out": orthogonalize(s["update"], steps=STEPS, coefficients=COEFFICIENTS,
                                     eps=UPDATE_EPS)}
    if case["kind"] == "embedding":
        out = token_embedding(s["ids"], s["weight"], scale=case["scale"],
                              padding_idx=_padding_id(case), dw_accumulator=s["accumulator"],
                              validate=False)
        if s["accumulator"] is not None:
            torch.autograd.grad(out, s["weight"], s["dout"], allow_unused=True)
            return {"out": out, "accumulator": s["accumulator"]}
        return {"out": out, "dweight": torch.autograd.grad(out, s["weight"], s["dout"])[0]}
    if case["residual"]:
        outs = residual_layer_norm(s["x"], s["residual"], s["weight"], s["bias"], eps=NORM_EPS,
                                   block_scale=case["block_scale"],
                                   residual_scale=case["residual_scale"])
        out, ups = dict(zip(("normed", "residual"), outs)), ("dnormed", "dresidual")
    else:
        outs = [layer_norm(s["x"], s["weight"], s["bias"], eps=NORM_EPS)]
        out, ups = {"normed": outs[0]}, ("dnormed",)
    if case["direction"] == "train":
        names = [n for n in ("x", "residual", "weight", "bias") if s[n] is not None]
        grads = torch.autograd.grad(outs, [s[n] for n in names], [s[u] for u in ups])
        out.update({"d" + n: g for n, g in zip(names, grads)})
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"embedding": _plain_embedding, "layer_norm": _plain_layer_norm,
            "orthogonalize": _plain_orthogonalize}[state["case"]["kind"]](state)


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "orthogonalize":
        m, n, batch = case["m"], case["n"], case["batch"]
        return {"bytes": 2 * es * batch * m * n, "flops": batch * _update_flops(m, n)}
    T, H = case["T"], case["H"]
    if case["kind"] == "embedding":
        V, looked = case["V"], T - case["padding"]
        # rows of the weight that some token asks for, on average
        rows = float((1.0 - torch.exp(looked * torch.log1p(-_zipf(V).clamp(max=1 - 1e-12)))).sum())
        gradient = 2 * 4 * rows * H if case["gradient"] == "accumulate" else es * V * H
        ids = T * (8 if case["ids"] == "int64" else 4)
        return {"bytes": ids + es * H * (rows + T + looked) + gradient, "flops": 3 * T * H}
    train = case["direction"] == "train"
    # x, the residual and the upstream gradients in; outputs and gradients out
    tensors = (8 if train else 4) if case["residual"] else (4 if train else 2)
    return {"bytes": tensors * T * H * es, "flops": (24 if train else 10) * T * H}


def _exact_embedding(case, s):
    ids = s["ids"].long()
    at = s["weight"].detach().double().requires_grad_(True)
    out = case["scale"] * torch.nn.functional.embedding(ids, at, padding_idx=_padding_id(case))
    (grad,) = torch.autograd.grad(out, at, s["dout"].double())
    out = out.detach()
    if s["accumulator"] is not None:
        return {"out": out, "accumulator": grad.add_(s["accumulator"])}
    return {"out": out, "dweight": grad}


def _exact_layer_norm(case, s):
    train = case["direction"] == "train"
    names = [n for n in ("x", "residual", "weight", "bias") if s[n] is not None]
    at = {n: s[n].detach().double().requires_grad_(train) for n in names}
    total = at["x"]
    if case["residual"]:
        total = case["residual_scale"] * at["residual"] + case["block_scale"] * total
    var, mean = torch.var_mean(total, -1, correction=0, keepdim=True)
    normed = (total - mean) / torch.sqrt(var + NORM_EPS) * at["weight"]
    if case["bias"]:
        normed = normed + at["bias"]
    out = {"normed": normed.detach()}
    outs, ups = [normed], ["dnormed"]
    if case["residual"]:
        out["residual"] = total.detach()
        outs.append(total)
        ups.append("dresidual")
    if train:
        grads = torch.autograd.grad(outs, [at[n] for n in names], [s[u].double() for u in ups])
        grads = {"d" + n: g for n, g in zip(names, grads)}
        order = ["dweight"] + (["dbias"] if case["bias"] else []) + \
            (["dresidual"] if case["residual"] else []) + ["dx"]
        out.update({n: grads[n] for n in order})
    return out


def _exact_orthogonalize(case, s):
    a, b, c = COEFFICIENTS
    stack = s["update"].reshape(-1, case["m"], case["n"])
    out = torch.empty(stack.shape, dtype=torch.float64, device="cuda")
    for k in range(len(stack)):
        x = stack[k].double()
        if case["m"] > case["n"]:
            x = x.T.contiguous()
        x = x / (torch.sqrt((x * x).sum()) + UPDATE_EPS)
        one = torch.eye(x.shape[0], dtype=torch.float64, device="cuda")
        for _ in range(STEPS):
            g = x @ x.T
            x = (a * one + g @ (b * one + c * g)) @ x
        out[k] = x.T if case["m"] > case["n"] else x
    return {"out": out.reshape(s["update"].shape)}


def exact(case, seed):
    return {"embedding": _exact_embedding, "layer_norm": _exact_layer_norm,
            "orthogonalize": _exact_orthogonalize}[case["kind"]](case, prepare(case, seed))
