"""The operators for adapting a frozen shift network, as cases that can be timed: low-rank adapters of many requests
beside a shared projection (serving and training), softmax cross entropy over a large vocabulary without its logits
(each row's loss alone, and the mean with its gradients), and the global norm of many gradients with their clipping.

Each case runs either in plain form (elementary torch operations in 32 bits, rounded once at the end) or, where ``own``
is true, through this package.  Sizes are those of the package's layers (512 ... 4096 wide linear layers, 1000-way
heads) and generic ones for vocabularies and batches."""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # One token of one request beside the hidden layer of the 784-512-512-10 network: latency is all there is.
        dict(name="adapters_m1_k512_n512_r8", kind="adapters", rows=1, k=512, n=512, rank=8, count=4, x="f32", w="f32",
             layout="tokens", train=False),
        # A decoding batch, one token a request, almost every one with an adapter of its own; the layer's fp32 in and out.
        dict(name="adapters_m64_k4096_n4096_r16", kind="adapters", rows=64, k=4096, n=4096, rank=16, count=64, x="f32",
             w="bf16", layout="tokens", train=False),
        # Prompts of several requests, ragged lengths, some requests without an adapter.
        dict(name="adapters_m8192_k2048_n2048_r64", kind="adapters", rows=8192, k=2048, n=2048, rank=64, count=12, x="bf16",
             w="bf16", layout="requests", train=False),
        # Sizes nothing is a multiple of anything, 16-bit floats, a rank of 5, rows of requests interleaved.
        dict(name="adapters_m1777_k1001_n777_r5", kind="adapters", rows=1777, k=1001, n=777, rank=5, count=9, x="f16", w="f16",
             layout="tokens", train=False),
        # A training step of four adapters at once in fp32, as the layers' own activations are: output and all gradients.
        dict(name="adapters_train_m4096_k4096_n4096_r32", kind="adapters", rows=4096, k=4096, n=4096, rank=32, count=4, x="f32",
             w="f32", layout="requests", train=True),
        # Evaluation of a 1000-way head on a few rows: each row's loss.
        dict(name="loss_n16_d512_v1000", kind="loss", rows=16, d=512, v=1000, x="bf16", train=False),
        # Scoring one long text: each token's loss, over a vocabulary of ordinary size.
        dict(name="loss_n2048_d1024_v32000", kind="loss", rows=2048, d=1024, v=32000, x="bf16", train=False),
        # A training step at odd sizes in 16-bit floats.
        dict(name="loss_train_n777_d520_v10007", kind="loss", rows=777, d=520, v=10007, x="f16", train=True),
        # A training step over the largest vocabulary, at full width.
        dict(name="loss_train_n8192_d4096_v131072", kind="loss", rows=8192, d=4096, v=131072, x="bf16", train=True),
        # Gradients of the adapters of a small network: few tensors, latency.
        dict(name="clip_t8_e65536_f32", kind="clip", tensors=8, most=65536, ragged=False, x="f32"),
        # All gradients of a convolution network as ResNet-18 has them in number: many sizes from a bias's on, odd ones, two types.
        dict(name="clip_t122_e2359296_mixed", kind="clip", tensors=122, most=2359296, ragged=True, x="mixed"),
        # Gradients of large 16-bit layers, far beyond the caches.
        dict(name="clip_t64_e16777216_bf16", kind="clip", tensors=64, most=16777216, ragged=False, x="bf16"),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _width(rng):
    step = rng.choice([1, 40, 320])   # any width, and multiples of a vector and of a tile's row
    return step * _log(rng, -(-64 // step), 4096 // step)


def draw(rng):
    kind = rng.choice(["adapters", "adapters", "adapters", "loss", "loss", "loss", "clip", "clip"])
    if kind == "adapters":
        x = rng.choice(["f32", "f32", "bf16", "f16"])
        train = rng.random() < 0.35
        return dict(kind=kind, rows=_log(rng, 1, 8192), k=_width(rng), n=_width(rng), rank=rng.choice([4, 5, 8, 16, 16, 24, 32, 64]),
                    count=_log(rng, 1, 64), x=x, w="bf16" if x == "f32" and not train and rng.random() < 0.5 else x,
                    layout=rng.choice(["tokens", "requests"]), train=train)
    if kind == "loss":
        while True:
            c = dict(kind=kind, rows=_log(rng, 1, 8192), d=_width(rng),
                     v=_log(rng, 100, 131072), x=rng.choice(["bf16", "bf16", "f16"]), train=rng.random() < 0.6)
            if work(c)["flops"] <= 1e13:
                return c
    c = dict(kind=kind, tensors=_log(rng, 1, 400), most=_log(rng, 64, 16777216), ragged=rng.random() < 0.7,
             x=rng.choice(["f32", "bf16", "f16", "mixed"]))
    c["most"] = min(c["most"], (1 << 29) // c["tensors"])
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _row_adapters(case, g):
    """Adapter of every row, -1 for none: one request a row, or requests of ragged lengths one behind another."""
    rows, count = case["rows"], case["count"]
    pick = lambda n: torch.randint(-1 if n > 1 else 0, count, (n,), generator=g, device="cuda", dtype=torch.int32)  # noqa: E731
    if case["layout"] == "tokens":
        return pick(rows)
    requests = max(1, min(rows, 2 * count))
    cuts = torch.randint(0, rows, (requests,), generator=g, device="cuda")
    request = (torch.arange(rows, device="cuda")[:, None] >= cuts.sort().values[None, 1:]).sum(1)
    return pick(requests)[request].contiguous()


def _clip_tensors(case, g):
    """Shapes as (elements, type): matrices, rows and single values; their number and sizes come from the case alone."""
    sizes = [case["most"]] * case["tensors"]
    if case["ragged"]:   # every third a bias, the others spread over the powers below the largest
        sizes = [max(1, min(case["most"], 1 + (i * 37) % 1000 if i % 3 == 0 else case["most"] // (1 + (i * i) % 23) - i % 7))
                 for i in range(case["tensors"])]
    kinds = [("f32" if i % 2 else "bf16") if case["x"] == "mixed" else case["x"] for i in range(case["tensors"])]
    return sizes, kinds


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "adapters":
        rows, k, n, r, count = (case[e] for e in ("rows", "k", "n", "rank", "count"))
        xt, wt = _TYPES[case["x"]], _TYPES[case["w"]]
        s = dict(case=case, ids=_row_adapters(case, g), x=_normal(g, rows, k).to(xt), base=_normal(g, rows, n).to(xt),
                 # trained adapters: a down projection as it was drawn, an up projection that has left zero
                 down=(_normal(g, count, r, k) / math.sqrt(k)).to(wt), up=(_normal(g, count, r, n) / math.sqrt(r)).to(wt),
                 scale=torch.rand(count, generator=g, device="cuda") * 2 + 0.25)
        if case["train"]:
            s["grad"] = (_normal(g, rows, n) * 0.1).to(xt)
        if own:   # one plan serves every layer of a batch
            from deepshift_b200 import adapters
            s["plan"] = adapters.plan_rows(s["ids"], count)
            if case["train"]:
                for e in ("x", "down", "up"):
                    s[e].requires_grad_(True)
        return s
    if case["kind"] == "loss":
        rows, d, v = case["rows"], case["d"], case["v"]
        t = _TYPES[case["x"]]
        weight = _normal(g, v, d).mul_(2 / math.sqrt(d)).to(t)
        # frequent tokens first, and hidden states that know most of their targets to some degree
        target = (torch.rand(rows, generator=g, device="cuda") ** 3 * v).long().clamp_(max=v - 1)
        know = torch.rand(rows, 1, generator=g, device="cuda") * 1.5
        hidden = (_normal(g, rows, d) + know * weight[target].float()).to(t)
        if rows > 1:   # padding and prompts do not count
            target[torch.rand(rows, generator=g, device="cuda") < 0.15] = -100
        s = dict(case=case, hidden=hidden, weight=weight, target=target)
        if own and case["train"]:
            s["hidden"].requires_grad_(True)
            s["weight"].requires_grad_(True)
        return s
    sizes, kinds = _clip_tensors(case, g)
    s = dict(case=case, grads=[], out=[], flat={})
    for t in sorted(set(kinds)):
        of = [n for n, e in zip(sizes, kinds) if e == t]
        s["flat"][t] = torch.empty(sum(of), device="cuda", dtype=_TYPES[t])
    at = dict.fromkeys(s["flat"], 0)
    total = 0.0
    for i, (n, t) in enumerate(zip(sizes, kinds)):
        std = 10.0 ** -(1 + i % 4)   # layers' gradients differ by orders of magnitude
        grad = torch.empty(n, device="cuda", dtype=_TYPES[t]).normal_(0, std, generator=g)
        s["grads"].append(grad.view(n // 64, 64) if n % 64 == 0 else grad)
        out = s["flat"][t][at[t]:at[t] + n]
        s["out"].append(out.view(n // 64, 64) if n % 64 == 0 else out)
        at[t] += n
        total += n * std * std
    s["max_norm"] = 0.3 * math.sqrt(total)   # the clipping takes effect
    return s


# ------------------------------------------------------------------------------------------------ one pass
def _plain_adapters(s):
    x, down, up = s["x"].float(), s["down"].float(), s["up"].float()
    count, r, k = down.shape
    ids = s["ids"].long()
    mine = (ids[:, None] == torch.arange(count, device=ids.device)).float() * s["scale"]         # [rows, count]
    every = (x @ down.reshape(count * r, k).T).reshape(-1, count, r)
    h = (every * mine[:, :, None]).reshape(-1, count * r)
    y = (s["base"].float() + h @ up.reshape(count * r, -1)).to(s["base"].dtype)
    if not s["case"]["train"]:
        return y
    grad = s["grad"].float()
    dh = ((grad @ up.reshape(count * r, -1).T).reshape(-1, count, r) * mine[:, :, None]).reshape(-1, count * r)
    return dict(y=y, x=(dh @ down.reshape(count * r, k)).to(s["x"].dtype),
                down=(dh.T @ x).reshape(down.shape).to(s["down"].dtype), up=(h.T @ grad).reshape(up.shape).to(s["up"].dtype))


def _plain_loss(s):
    hidden, weight, target = s["hidden"].float(), s["weight"].float(), s["target"]
    logits = hidden @ weight.T
    top = logits.max(1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    valid = target >= 0
    at = target.clamp(min=0)[:, None]
    each = (top + torch.log(total) - logits.gather(1, at))[:, 0]
    each = torch.where(valid, each, torch.zeros_like(each))
    if not s["case"]["train"]:
        return each
    count = valid.sum()
    loss = each.sum() / count
    g = e / total
    g.scatter_add_(1, at, torch.full_like(each, -1.0)[:, None])
    g = g * (valid / count.clamp(min=1))[:, None]
    return dict(loss=loss, hidden=(g @ weight).to(s["hidden"].dtype), weight=(g.T @ hidden).to(s["weight"].dtype))


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return dict(norm=norm, **{t: torch.cat([(g.float() * factor).to(g.dtype).reshape(-1) for g in s["grads"] if g.dtype == _TYPES[t]])
                              for t in s["flat"]})


def run(s):
    case = s["case"]
    if not own:
        return {"adapters": _plain_adapters, "loss": _plain_loss, "clip": _plain_clip}[case["kind"]](s)
    if case["kind"] == "adapters":
        from deepshift_b200 import adapters
        y = adapters.apply(s["x"], s["down"], s["up"], s["scale"], s["plan"], base=s["base"])
        if not case["train"]:
            return y
        dx, ddown, dup = torch.autograd.grad(y, (s["x"], s["down"], s["up"]), s["grad"])
        return dict(y=y, x=dx, down=ddown, up=dup)
    if case["kind"] == "loss":
        from deepshift_b200 import losses
        if not case["train"]:
            return losses.linear_cross_entropy(s["hidden"], s["weight"], s["target"], reduction="none")
        loss = losses.linear_cross_entropy(s["hidden"], s["weight"], s["target"])
        dh, dw = torch.autograd.grad(loss, (s["hidden"], s["weight"]))
        return dict(loss=loss, hidden=dh, weight=dw)
    from deepshift_b200 import gradients
    norm = gradients.clip_norm(s["grads"], s["max_norm"], out=s["out"])
    return dict(norm=norm, **s["flat"])


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    if case["kind"] == "adapters":
        rows, k, n, r = (case[e] for e in ("rows", "k", "n", "rank"))
        bx, bw = (2 if case[e] != "f32" else 4 for e in ("x", "w"))
        weights = min(case["count"], rows if case["layout"] == "tokens" else 2 * case["count"]) * r * (k + n) * bw
        if case["train"]:   # x, base and the output's gradient in, output and x's gradient out, weights in, their gradients out
            return dict(bytes=rows * (2 * k + 3 * n) * bx + 2 * weights, flops=6 * rows * r * (k + n))
        return dict(bytes=rows * (k + 2 * n) * bx + weights, flops=2 * rows * r * (k + n))
    if case["kind"] == "loss":
        rows, d, v = case["rows"], case["d"], case["v"]
        once = (rows * d + v * d) * 2
        return dict(bytes=once * (2 if case["train"] else 1) + rows * 8, flops=2 * rows * d * v * (3 if case["train"] else 1))
    sizes, kinds = _clip_tensors(case, None)
    total = sum(n * (4 if t == "f32" else 2) for n, t in zip(sizes, kinds))
    return dict(bytes=2 * total, flops=3 * sum(sizes))


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "adapters":
        x, base, ids, scale = s["x"].detach().double(), s["base"].double(), s["ids"], s["scale"].double()
        down, up = s["down"].detach().double(), s["up"].detach().double()
        y, dx, ddown, dup = base.clone(), torch.zeros_like(x), torch.zeros_like(down), torch.zeros_like(up)
        for a in range(case["count"]):
            at = torch.nonzero(ids == a)[:, 0]
            if not len(at):
                continue
            h = torch.einsum("mk,rk->mr", x[at], down[a])
            y[at] += scale[a] * torch.einsum("mr,rn->mn", h, up[a])
            if case["train"]:
                grad = s["grad"][at].double()
                dh = scale[a] * torch.einsum("mn,rn->mr", grad, up[a])
                dx[at] = torch.einsum("mr,rk->mk", dh, down[a])
                ddown[a] = torch.einsum("mr,mk->rk", dh, x[at])
                dup[a] = scale[a] * torch.einsum("mr,mn->rn", h, grad)
        return dict(y=y, x=dx, down=ddown, up=dup) if case["train"] else y
    if case["kind"] == "loss":
        hidden, target = s["hidden"].detach().double(), s["target"]
        weight = s["weight"].detach().double()
        rows = int((target != -100).sum())
        each, dh, dw = hidden.new_zeros(case["rows"]), torch.zeros_like(hidden), torch.zeros_like(weight)
        for first in range(0, case["rows"], 1024):
            part = slice(first, min(case["rows"], first + 1024))
            live = torch.nonzero(target[part] != -100)[:, 0]
            if not len(live):
                continue
            logs = torch.log_softmax(torch.einsum("nd,vd->nv", hidden[part][live], weight), dim=1)
            t = target[part][live]
            each[part][live] = -logs[torch.arange(len(t), device=t.device), t]
            if case["train"]:
                p = logs.exp_()
                p[torch.arange(len(t), device=t.device), t] -= 1
                p /= rows
                dh[part][live] = p @ weight
                dw += p.T @ hidden[part][live]
        # every target ignored: no mean, and no gradient
        loss = each.sum() / rows if rows else each.sum() * math.nan
        return dict(loss=loss, hidden=dh, weight=dw) if case["train"] else each
    norm = math.sqrt(math.fsum(float(g.double().pow(2).sum()) for g in s["grads"]))
    factor = min(1.0, s["max_norm"] / (norm + 1e-6))
    return dict(norm=torch.tensor(norm, dtype=torch.float64),
                **{t: torch.cat([g.double().flatten() for g in s["grads"] if g.dtype == _TYPES[t]]) * factor for t in s["flat"]})
