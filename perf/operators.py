"""Cases, plain forms and exact values of the output head's operators: ``layer_norm``, ``dropout``,
``linear_log_softmax`` and ``linear_cross_entropy`` of ``waterfall_amd``.

A case names an operator, the padded batch ``[batch, time]`` it sees, the encoder's width ``dim``, the number of output
tokens ``vocab`` and the type of the activations.  ``train`` cases run the operator and its gradients.
"""
import math

import numpy as np
import torch

own = False

F = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------------
# the cases

def _case(name, op, batch, time, dim, dtype, train, vocab=0, params="", p=0.0, smoothing=0.0, reduction="mean", bias=True):
    return {"name": name, "op": op, "batch": batch, "time": time, "dim": dim, "vocab": vocab, "dtype": dtype,
            "params": params or dtype, "train": train, "p": p, "smoothing": smoothing, "reduction": reduction, "bias": bias}


def listed():
    return [
        # one frame of one stream: the norm of a streaming recogniser, a call that is all latency
        _case("norm_one_frame", "layer_norm", 1, 1, 512, "float32", False),
        # the benchmark's batch (32 utterances of 500 frames) under mixed precision: activations in bfloat16, weights in fp32
        _case("norm_batch", "layer_norm", 32, 500, 512, "bfloat16", True, params="float32"),
        # a long batch of wide features
        _case("norm_long", "layer_norm", 16, 3000, 1024, "float32", True),
        # the benchmark's batch of wide features on its way into the projection
        _case("dropout_batch", "dropout", 32, 500, 1024, "bfloat16", True, p=0.1),
        # an odd width and an odd batch in fp32
        _case("dropout_odd", "dropout", 7, 333, 515, "float32", True, p=0.25),
        # a chunk of four frames of one stream scored against a BPE vocabulary (serving)
        _case("log_softmax_chunk", "linear_log_softmax", 1, 4, 512, "bfloat16", False, vocab=5001),
        # character units, fp32 training
        _case("log_softmax_chars", "linear_log_softmax", 32, 500, 512, "float32", True, vocab=59),
        # the benchmark's batch and vocabulary, trained: the projection whose result the graph loss takes
        _case("log_softmax_batch", "linear_log_softmax", 32, 500, 512, "bfloat16", True, vocab=5001),
        # the targets of a small batch, odd sizes, fp32
        _case("entropy_small", "linear_cross_entropy", 8, 37, 257, "float32", True, vocab=5001, smoothing=0.1),
        # the benchmark's batch and vocabulary, frame targets
        _case("entropy_batch", "linear_cross_entropy", 32, 500, 512, "bfloat16", True, vocab=5001),
        # per-frame losses in half precision, two tokens per phone (10 001 outputs)
        _case("entropy_frames", "linear_cross_entropy", 16, 481, 768, "float16", True, vocab=10001, reduction="none"),
        # the largest vocabulary of the benchmark's topologies, a wide encoder
        _case("entropy_large", "linear_cross_entropy", 32, 500, 1024, "bfloat16", True, vocab=15001, smoothing=0.1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "dropout", "linear_log_softmax", "linear_cross_entropy"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    batch, time, dim = _log(rng, 1, 48), _log(rng, 1, 1500), _log(rng, 64, 1280)
    if rng.random() < 0.5:
        dim = max(64, dim // 64 * 64)
    c = {"op": op, "dtype": dtype, "params": dtype, "train": rng.random() < 0.7, "p": 0.0, "smoothing": 0.0,
         "reduction": "mean", "bias": rng.random() < 0.8, "vocab": 0}
    if op == "layer_norm":
        c["params"] = rng.choice([dtype, "float32"])
    elif op == "dropout":
        c["p"] = round(rng.uniform(0.02, 0.6), 3)
    else:
        c["vocab"] = _log(rng, 29, 15001)
        most = 16000 * 15001 * 1024 / (8 if dtype == "float32" else 1)      # multiplications of the largest listed case
        while batch * time * dim * c["vocab"] > most or batch * time > 24000:
            time = max(1, time // 2)
        if op == "linear_cross_entropy":
            c["smoothing"] = rng.choice([0.0, 0.1])
            c["reduction"] = rng.choice(["mean", "sum", "none"])
    c.update(batch=batch, time=time, dim=dim)
    return c


# ---------------------------------------------------------------------------------------------------------------------
# inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, T, D, V = case["batch"], case["time"], case["dim"], case["vocab"]
    dt, pt, train = F[case["dtype"]], F[case["params"]], case["train"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def leaf(t):
        return t.requires_grad_() if train else t

    s = {"case": case}
    if case["op"] in ("layer_norm", "dropout"):
        # an encoder's output: features of unlike scale and offset
        s["x"] = leaf((normal(B, T, D) * (0.5 + torch.rand(D, device="cuda", generator=g)) + 0.3 * normal(D)).to(dt))
        if train:
            s["g"] = normal(B, T, D).to(dt)
    else:
        s["x"] = leaf(normal(B, T, D).to(dt))                           # normalised features
        s["weight"] = leaf((normal(V, D) * (2.0 / math.sqrt(D))).to(dt))
        s["bias"] = leaf((0.5 * normal(V)).to(dt)) if case["bias"] else None
    if case["op"] == "layer_norm":
        s["weight"] = leaf((1.0 + 0.1 * normal(D)).to(pt))
        s["bias"] = leaf((0.1 * normal(D)).to(pt)) if case["bias"] else None
    elif case["op"] == "dropout":
        s["seed"] = int(torch.randint(0, 1 << 62, (1,), generator=torch.Generator().manual_seed(seed)))
    elif case["op"] == "linear_log_softmax":
        if train:
            # what a graph loss hands back: minus a numerator's posteriors, a few tokens per frame, nothing behind the end
            length = torch.randint(max(1, T * 3 // 4), T + 1, (B,), device="cuda", generator=g)
            there = torch.arange(T, device="cuda") < length[:, None]
            s["g"] = torch.softmax(6 * normal(B, T, V), -1).mul_(there[..., None]).neg_()
    else:
        # a padded batch: the frames behind an utterance's end have no target
        length = torch.randint(max(1, T * 3 // 4), T + 1, (B,), device="cuda", generator=g)
        t = torch.randint(0, V, (B, T), device="cuda", generator=g)
        s["targets"] = torch.where(torch.arange(T, device="cuda") < length[:, None], t, -1)
        if train:
            s["g"] = 0.5 + torch.rand(B, T, device="cuda", generator=g) if case["reduction"] == "none" else torch.ones((), device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass

def run(s):
    op, train = s["case"]["op"], s["case"]["train"]
    if own:
        y = _call(s)
        if not train:
            return {"y": y}
        names = [n for n in ("x", "weight", "bias") if s.get(n) is not None]
        return {"y": y.detach(), **{"d" + n: t for n, t in zip(names, torch.autograd.grad(y, [s[n] for n in names], s["g"]))}}
    with torch.no_grad():
        return _PLAIN[op](s)


def _call(s):
    import waterfall_amd as wf
    c = s["case"]
    if c["op"] == "layer_norm":
        return wf.layer_norm(s["x"], s["weight"], s["bias"])
    if c["op"] == "dropout":
        return wf.dropout(s["x"], c["p"], s["seed"])
    if c["op"] == "linear_log_softmax":
        return wf.linear_log_softmax(s["x"], s["weight"], s["bias"])
    return wf.linear_cross_entropy(s["x"], s["weight"], s["targets"], s["bias"], label_smoothing=c["smoothing"],
                                   reduction=c["reduction"])


def _norm(s):
    x, w = s["x"].float(), s["weight"].float()
    d = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((d * d).mean(-1, keepdim=True) + 1e-5)
    h = d * r
    y = h * w
    if s["bias"] is not None:
        y = y + s["bias"].float()
    out = {"y": y.to(s["x"].dtype)}
    if s["case"]["train"]:
        g = s["g"].float()
        gw = g * w
        dx = r * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
        out["dx"] = dx.to(s["x"].dtype)
        out["dweight"] = (g * h).sum((0, 1)).to(s["weight"].dtype)
        if s["bias"] is not None:
            out["dbias"] = g.sum((0, 1)).to(s["bias"].dtype)
    return out


def _mulhilo(a, m):
    """The two 32-bit halves of a * m, a in [0, 2^32) held in int64, m a number below 2^32."""
    lo16, hi16 = a & 0xFFFF, a >> 16
    low = lo16 * m                                # below 2^48
    high = hi16 * m + (low >> 16)                 # below 2^49
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def _philox(n, seed):
    """n 32-bit words of Philox4x32-7 (Salmon et al., Parallel random numbers: as easy as 1, 2, 3; 2011): the words of the
    counters 0, 1, 2, ... under the key `seed`."""
    i = torch.arange((n + 3) // 4, device="cuda", dtype=torch.int64)
    c0, c1, c2, c3 = i & 0xFFFFFFFF, i >> 32, torch.zeros_like(i), torch.zeros_like(i)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF
    for r in range(7):
        h0, l0 = _mulhilo(c0, 0xD2511F53)
        h1, l1 = _mulhilo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:n]


def _drop(s):
    x, p = s["x"], s["case"]["p"]
    kept = (_philox(x.numel(), s["seed"]) >= int(p * 4294967296.0)).reshape(x.shape)
    scale = 1.0 / (1.0 - p)
    out = {"y": torch.where(kept, x.float() * scale, 0.0).to(x.dtype)}
    if s["case"]["train"]:
        out["dx"] = torch.where(kept, s["g"].float() * scale, 0.0).to(x.dtype)
    return out


def _logits(s):
    z = s["x"].float().reshape(-1, s["case"]["dim"]) @ s["weight"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    return z, torch.logsumexp(z, -1, keepdim=True)


def _projection(s, dz, out):
    x = s["x"].float().reshape(-1, s["case"]["dim"])
    out["dx"] = (dz @ s["weight"].float()).reshape(s["x"].shape).to(s["x"].dtype)
    out["dweight"] = (dz.t() @ x).to(s["weight"].dtype)
    if s["bias"] is not None:
        out["dbias"] = dz.sum(0).to(s["bias"].dtype)
    return out


def _log_softmax(s):
    z, lse = _logits(s)
    lp = z - lse
    out = {"y": lp.reshape(s["x"].shape[:-1] + (s["case"]["vocab"],))}
    if s["case"]["train"]:
        g = s["g"].reshape(lp.shape)
        _projection(s, g - torch.exp(lp) * g.sum(-1, keepdim=True), out)
    return out


def _entropy(s):
    c, t = s["case"], s["targets"].reshape(-1)
    z, lse = _logits(s)
    there, at = t >= 0, t.clamp(min=0)[:, None]
    e = c["smoothing"]
    loss = lse[:, 0] - (1 - e) * z.gather(1, at)[:, 0]
    if e:
        loss = loss - e * z.mean(-1)
    loss = torch.where(there, loss, 0.0)
    n = there.sum()
    out = {"y": loss.reshape(s["targets"].shape) if c["reduction"] == "none" else loss.sum() if c["reduction"] == "sum" else loss.sum() / n}
    if c["train"]:
        g = s["g"].reshape(-1) if c["reduction"] == "none" else s["g"] if c["reduction"] == "sum" else s["g"] / n
        g = torch.where(there, g, 0.0)[:, None]
        dz = torch.exp(z - lse) - e / c["vocab"]
        dz.scatter_add_(1, at, torch.full_like(at, -(1 - e), dtype=dz.dtype))
        _projection(s, dz * g, out)
    return out


_PLAIN = {"layer_norm": _norm, "dropout": _drop, "linear_log_softmax": _log_softmax, "linear_cross_entropy": _entropy}


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    n, D, V = case["batch"] * case["time"], case["dim"], case["vocab"]
    size = {"float32": 4, "bfloat16": 2, "float16": 2}
    e, pe, train = size[case["dtype"]], size[case["params"]], case["train"]
    par = D * pe * (2 if case["bias"] else 1)
    if case["op"] == "layer_norm":
        return {"bytes": 2 * n * D * e + par + (2 * n * D * e + par if train else 0), "flops": n * D * (8 + (12 if train else 0))}
    if case["op"] == "dropout":
        return {"bytes": (4 if train else 2) * n * D * e, "flops": n * D * (2 if train else 1)}
    par = (V * D + (V if case["bias"] else 0)) * e
    box = 4 * n * V if case["op"] == "linear_log_softmax" else 12 * n
    # training: the inputs once, the gradient that comes in once (a box of its own for log-probabilities), the outputs once
    return {"bytes": n * D * e * (2 if train else 1) + par * (2 if train else 1) + box * (2 if train and case["op"] == "linear_log_softmax" else 1),
            "flops": 2 * n * V * D * (3 if train else 1)}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach().double().requires_grad_()
    leaves = {"x": x}
    for name in ("weight", "bias"):
        if s.get(name) is not None:
            leaves[name] = s[name].detach().double().requires_grad_()
    op = case["op"]
    if op == "layer_norm":
        var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
        y = (x - mean) / (var + 1e-5).sqrt() * leaves["weight"] + leaves.get("bias", 0.0)
    elif op == "dropout":
        keep = torch.from_numpy(_words(x.numel(), s["seed"]) >= np.uint64(math.floor(case["p"] * 2.0 ** 32))).cuda().reshape(x.shape)
        y = torch.where(keep, x / (1 - case["p"]), torch.zeros_like(x))
    else:
        y = torch.log_softmax(torch.matmul(x, leaves["weight"].mT) + leaves.get("bias", 0.0), -1)
        if op == "linear_cross_entropy":
            there = s["targets"] >= 0
            e = case["smoothing"]
            one = torch.nn.functional.one_hot(s["targets"].clamp(min=0), case["vocab"])
            loss = -((1 - e) * (y * one).sum(-1) + e * y.mean(-1)) * there
            y = loss if case["reduction"] == "none" else loss.sum() / (there.sum() if case["reduction"] == "mean" else 1)
            del one
    out = {"y": y.detach()}
    if case["train"]:
        for name, t in zip(leaves, torch.autograd.grad(y, list(leaves.values()), s["g"].double())):
            out["d" + name] = t
    return out


def _words(n, seed):
    """The generator's words by unsigned 64-bit arithmetic."""
    low, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = np.zeros((4, (n + 3) // 4), np.uint64)
    c[0] = np.arange(c.shape[1], dtype=np.uint64)
    c[1], c[0] = c[0] >> sh, c[0] & low
    key = [seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32]
    for _ in range(7):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = np.stack([(b >> sh) ^ c[1] ^ np.uint64(key[0]), b & low, (a >> sh) ^ c[3] ^ np.uint64(key[1]), a & low])
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    return c.T.reshape(-1)[:n]
