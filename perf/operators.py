"""Cases for measuring the vocabulary operators around the sampler: the LM head with 4-bit weights, the embedding
lookup and its gradient, token log-probabilities with their gradient, and the clipped policy loss with its gradient.

With `own` false, `run` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once
at the end); with `own` true it makes the calls that a user makes of the framework.  `exact` is the definition in 64
bits, written apart from the plain form."""
import math

import torch

own = False

BF16, F32 = "bf16", "f32"
_T = {BF16: torch.bfloat16, F32: torch.float32}
_SIZE = {BF16: 2, F32: 4}


def listed():
    return [
        # a single request's decode step: the 152k vocabulary's head in 4 bits, one hidden row
        dict(name="w4 head, one row", op="w4", B=1, V=151936, d=2048, g=128, stype=BF16, zeros=False, out=F32),
        # the mixed continuous batch of 64 rows, logits in bf16 for the sampler
        dict(name="w4 head, 64 rows", op="w4", B=64, V=151936, d=2048, g=128, stype=BF16, zeros=True, out=BF16),
        # a codec head of a depth loop: a small vocabulary, fine groups, f32 scales; latency counts
        dict(name="w4 codec head", op="w4", B=16, V=4099, d=1024, g=32, stype=F32, zeros=True, out=F32),
        # a large decode batch on a wide model: more products than bytes
        dict(name="w4 head, 200 rows", op="w4", B=200, V=128256, d=4096, g=64, stype=BF16, zeros=False, out=BF16),
        # log-probabilities of the ids that a decode step of 64 rows sampled
        dict(name="logprobs of a step", op="logp", N=64, V=151936, dtype=BF16, temperature=1.0, masked=0.0),
        # the gradient of a loss on log-probabilities (odd vocabulary, f32, temperature)
        dict(name="logprobs gradient", op="logp_grad", N=1000, V=32001, dtype=F32, temperature=0.7, masked=0.0),
        # one policy update over 4096 sampled tokens
        dict(name="policy loss, 4096 tokens", op="policy", N=4096, V=151936, dtype=BF16, temperature=1.0, masked=0.0,
             kl=0.04, ref=True),
        # a short batch in f32 whose vocabulary is constrained (a quarter of the logits are -inf)
        dict(name="policy loss, 257 tokens", op="policy", N=257, V=128256, dtype=F32, temperature=0.6, masked=0.25,
             kl=0.0, ref=False),
        # the next step's input: 64 sampled ids looked up in the tied 4-bit table
        dict(name="w4 lookup of a step", op="embed_w4", N=64, V=151936, d=2048, g=128, stype=BF16, zeros=False,
             out=BF16),
        # a prompt's lookup with the square root of the width as its scale
        dict(name="lookup of a prompt", op="embed", N=16384, V=128256, d=2048, dtype=BF16, out=BF16),
        # the embedding's gradient of one update, dense, over Zipf-distributed ids
        dict(name="lookup gradient", op="embed_grad", N=16384, V=151936, d=2048, dtype=BF16, out=BF16, base=False),
        # a codec table's gradient, added to the tied head's: few rows, many tokens of each
        dict(name="codec lookup gradient", op="embed_grad", N=30011, V=4099, d=1024, dtype=BF16, out=F32, base=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("w4", "w4", "logp", "logp_grad", "policy", "policy", "embed_w4", "embed", "embed_grad", "embed_grad"))
    V = _log(rng, 1000, 156940)
    dtype, out = rng.choice((BF16, F32)), rng.choice((BF16, F32))
    if op == "w4":
        return dict(op=op, B=_log(rng, 1, 256), V=V, d=128 * _log(rng, 4, 32), g=rng.choice((32, 64, 128)),
                    stype=rng.choice((BF16, F32)), zeros=rng.random() < 0.5, out=out)
    if op == "embed_w4":
        return dict(op=op, N=_log(rng, 1, 8192), V=V, d=128 * _log(rng, 4, 32), g=rng.choice((32, 64, 128)),
                    stype=rng.choice((BF16, F32)), zeros=rng.random() < 0.5, out=out)
    if op == "embed":
        return dict(op=op, N=_log(rng, 1, 32768), V=V, d=_log(rng, 500, 4096), dtype=dtype, out=out)
    if op == "embed_grad":
        return dict(op=op, N=_log(rng, 1, 32768), V=V, d=_log(rng, 500, 4096), dtype=dtype, out=out,
                    base=rng.random() < 0.5)
    N = max(1, min(_log(rng, 1, 4096), 600_000_000 // (V * (2 if dtype == F32 else 1))))
    c = dict(op=op, N=N, V=V, dtype=dtype, temperature=rng.choice((1.0, 0.6, 1.3)), masked=rng.choice((0.0, 0.0, 0.25)))
    if op == "policy":
        c.update(kl=rng.choice((0.0, 0.04)), ref=True)
    return c


# ------------------------------------------------------------------ inputs


def _weights(c, gen):
    """4-bit weights as a group quantiser leaves them: codes bunched about the zero point, positive scales."""
    V, d, g = c["V"], c["d"], c["g"]
    codes = torch.randn(V, d // 2, 2, device="cuda", generator=gen).mul_(2.7).add_(8).round_().clamp_(0, 15).to(torch.uint8)
    packed = codes[..., 0] | (codes[..., 1] << 4)
    scales = (torch.rand(V, d // g, device="cuda", generator=gen) + 0.5) / math.sqrt(d)
    zeros = None
    if c["zeros"]:
        zeros = torch.randint(5, 12, (V, d // g), device="cuda", generator=gen, dtype=torch.uint8)
    return dict(packed=packed, scales=scales.to(_T[c["stype"]]), zeros=zeros)


def _ids(N, V, gen):
    """Zipf-like ids (the low ids are the frequent ones), about one in forty a padding row (-1)."""
    u = torch.rand(N, device="cuda", generator=gen, dtype=torch.float64)
    ids = (torch.exp(u * math.log(V + 1)).long() - 1).clamp_(0, V - 1)
    pad = torch.rand(N, device="cuda", generator=gen) < 0.025
    pad[0] = False
    return torch.where(pad, -1, ids)


def _logits(c, gen):
    N, V = c["N"], c["V"]
    x = torch.randn(N, V, device="cuda", generator=gen).mul_(3)
    k = max(1, V // 200)  # spikes, as in the sampler's mixed workload
    at = torch.randint(0, V, (N, k), device="cuda", generator=gen)
    x.scatter_add_(1, at, 4 + 6 * torch.rand(N, k, device="cuda", generator=gen))
    # what a rollout samples: the ids of the largest of a few random candidates and one of the spikes
    cand = torch.cat([at[:, :1], torch.randint(0, V, (N, 7), device="cuda", generator=gen)], 1)
    ids = cand.gather(1, x.gather(1, cand).argmax(1, keepdim=True))
    if c["masked"]:  # ids that a grammar disallows; the sampled one is allowed
        keep = x.gather(1, ids)
        x.masked_fill_(torch.rand(N, V, device="cuda", generator=gen) < c["masked"], float("-inf"))
        x.scatter_(1, ids, keep)
    return x.to(_T[c["dtype"]]), ids[:, 0]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(c=c)
    if c["op"] == "w4":
        s.update(_weights(c, gen))
        s["hidden"] = torch.randn(c["B"], c["d"], device="cuda", generator=gen).to(torch.bfloat16)
    elif c["op"] == "embed_w4":
        s.update(_weights(c, gen))
        s["ids"] = _ids(c["N"], c["V"], gen)
        s["scale"] = math.sqrt(c["d"])
    elif c["op"] == "embed":
        s["table"] = torch.randn(c["V"], c["d"], device="cuda", generator=gen).mul_(0.02).to(_T[c["dtype"]])
        s["ids"] = _ids(c["N"], c["V"], gen)
        s["scale"] = math.sqrt(c["d"])
    elif c["op"] == "embed_grad":
        s["dout"] = torch.randn(c["N"], c["d"], device="cuda", generator=gen).mul_(0.01).to(_T[c["dtype"]])
        s["ids"] = _ids(c["N"], c["V"], gen)
        s["scale"] = math.sqrt(c["d"])
        s["base"] = None
        if c["base"]:
            s["base"] = torch.randn(c["V"], c["d"], device="cuda", generator=gen).mul_(0.1).to(_T[c["out"]])
    else:
        s["logits"], s["ids"] = _logits(c, gen)
        N, T = c["N"], c["temperature"]
        step = max(1, 100_000_000 // c["V"])
        lse = torch.cat([torch.logsumexp(s["logits"][i:i + step].double() / T, 1) for i in range(0, N, step)])
        logp = s["logits"].gather(1, s["ids"][:, None])[:, 0].double() / T - lse
        if c["op"] == "logp_grad":
            s["lse"] = lse.float()
            s["dlogp"] = torch.randn(N, device="cuda", generator=gen) / N
        if c["op"] == "policy":
            noise = 0.15 * torch.randn(N, device="cuda", generator=gen, dtype=torch.float64)
            # no token sits within 1e-3 of the clip's border, where the gradient jumps
            r = torch.exp(noise)
            near = ((r - 0.8).abs() < 1e-3) | ((r - 1.2).abs() < 1e-3)
            s["old"] = (logp - noise - 0.02 * near).float()
            s["adv"] = torch.randn(N, device="cuda", generator=gen)
            s["ref"] = (logp + 0.3 * torch.randn(N, device="cuda", generator=gen)).float() if c["ref"] else None
            s["weights"] = torch.full((N,), 1.0 / N, device="cuda")
            pad = torch.rand(N, device="cuda", generator=gen) < 0.05  # the batch's padding
            pad[0] = False
            s["ids"] = torch.where(pad, -1, s["ids"])
    return s


# ------------------------------------------------------------------ one pass


def run(state):
    s, c = state, state["c"]
    if own:
        return _calls(s, c)
    if c["op"] == "w4":
        w = _plain_dequant(s["packed"], s["scales"], s["zeros"])
        return (s["hidden"].float() @ w.t()).to(_T[c["out"]])
    if c["op"] == "embed_w4":
        at = s["ids"].clamp(min=0)
        rows = _plain_dequant(s["packed"][at], s["scales"][at], None if s["zeros"] is None else s["zeros"][at])
        return (rows * s["scale"] * (s["ids"] >= 0)[:, None]).to(_T[c["out"]])
    if c["op"] == "embed":
        rows = s["table"][s["ids"].clamp(min=0)].float()
        return (rows * s["scale"] * (s["ids"] >= 0)[:, None]).to(_T[c["out"]])
    if c["op"] == "embed_grad":
        grad = torch.zeros(c["V"], c["d"], device="cuda")
        valid = (s["ids"] >= 0).float()[:, None]
        grad.index_add_(0, s["ids"].clamp(min=0), s["dout"].float() * valid)
        grad *= s["scale"]
        if s["base"] is not None:
            grad += s["base"]
        return grad.to(_T[c["out"]])
    return _plain_rows(s, c)


def _plain_dequant(packed, scales, zeros):
    q = torch.stack([packed & 15, packed >> 4], 2).float().view(packed.shape[0], scales.shape[1], -1)
    z = 8.0 if zeros is None else zeros.float()[:, :, None]
    return ((q - z) * scales.float()[:, :, None]).view(packed.shape[0], -1)


def _plain_rows(s, c):
    """Log-probabilities, their gradient or the policy loss: the rows in 32 bits, each row's scalars in 64 (a ratio
    and a KL term lose what matters when 32 bits hold the log-probabilities they are differences of)."""
    T = c["temperature"]
    valid = s["ids"] >= 0
    at = s["ids"].clamp(min=0)[:, None]
    x = s["logits"].float()
    m = x.max(1, keepdim=True).values
    chosen = x.gather(1, at)[:, 0].double()
    if c["op"] == "logp_grad":
        d = s["dlogp"] * valid / T
        grad = torch.exp(x / T - s["lse"][:, None]) * -d[:, None]
        grad.scatter_add_(1, at, d[:, None])
        return grad.to(_T[c["dtype"]])
    e = torch.exp((x - m) / T)
    total = e.sum(1, keepdim=True)
    lse = (m.double() / T + total.double().log())[:, 0]
    logp = torch.where(valid, chosen / T - lse, 0.0)
    if c["op"] == "logp":
        return dict(logp=logp.float(), lse=lse.float())
    r = torch.exp(logp - s["old"].double())
    a = s["adv"].double()
    clipped = r.clamp(0.8, 1.2)
    loss = -torch.minimum(r * a, clipped * a)
    dlogp = torch.where(r * a <= clipped * a, -r * a, 0.0)
    if s["ref"] is not None:
        k = s["ref"].double() - logp
        loss = loss + c["kl"] * (torch.expm1(k) - k)
        dlogp = dlogp - c["kl"] * torch.expm1(k)
    loss = torch.where(valid, loss, 0.0)
    d = (torch.where(valid, dlogp * s["weights"], 0.0) / T).float()[:, None]
    grad = e / total * -d
    grad.scatter_add_(1, at, d)
    return dict(loss=loss.float(), logp=logp.float(), dlogits=grad.to(_T[c["dtype"]]))


def _calls(s, c):
    """The framework's own calls."""
    from mstar_rs_b200 import kernel

    if c["op"] == "w4":
        return kernel.lmhead_logits_w4(s["hidden"], s["packed"], s["scales"], zeros=s["zeros"], dtype=_T[c["out"]])
    if c["op"] == "embed_w4":
        return kernel.embed_tokens_w4(s["ids"], s["packed"], s["scales"], zeros=s["zeros"], scale=s["scale"],
                                      dtype=_T[c["out"]])
    if c["op"] == "embed":
        return kernel.embed_tokens(s["ids"], s["table"], scale=s["scale"], dtype=_T[c["out"]])
    if c["op"] == "embed_grad":
        return kernel.embed_tokens_grad(s["ids"], s["dout"], c["V"], scale=s["scale"], base=s["base"],
                                        dtype=_T[c["out"]])
    if c["op"] == "logp":
        logp, lse = kernel.token_logprobs(s["logits"], s["ids"], temperature=c["temperature"])
        return dict(logp=logp, lse=lse)
    if c["op"] == "logp_grad":
        return kernel.token_logprobs_grad(s["logits"], s["ids"], s["lse"], s["dlogp"], temperature=c["temperature"])
    loss, logp, dlogits = kernel.policy_loss(s["logits"], s["ids"], s["old"], s["adv"], ref_logp=s["ref"],
                                             weights=s["weights"], temperature=c["temperature"], clip_low=0.2,
                                             clip_high=0.2, kl_coef=c["kl"])
    return dict(loss=loss, logp=logp, dlogits=dlogits)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c = case
    if c["op"] in ("w4", "embed_w4"):
        per_row = c["d"] // 2 + c["d"] // c["g"] * (_SIZE[c["stype"]] + (1 if c["zeros"] else 0))
        if c["op"] == "embed_w4":
            n = c["N"]
            return dict(bytes=n * (8 + per_row + c["d"] * _SIZE[c["out"]]), flops=2 * n * c["d"])
        B, V, d = c["B"], c["V"], c["d"]
        return dict(bytes=V * per_row + B * d * 2 + B * V * _SIZE[c["out"]], flops=2 * B * V * d)
    if c["op"] == "embed":
        return dict(bytes=c["N"] * (8 + c["d"] * (_SIZE[c["dtype"]] + _SIZE[c["out"]])), flops=c["N"] * c["d"])
    if c["op"] == "embed_grad":
        table = c["V"] * c["d"] * _SIZE[c["out"]]
        return dict(bytes=c["N"] * (8 + c["d"] * _SIZE[c["dtype"]]) + table * (2 if c["base"] else 1),
                    flops=2 * c["N"] * c["d"])
    row = c["V"] * _SIZE[c["dtype"]]
    passes = 1 if c["op"] == "logp" else 2
    return dict(bytes=c["N"] * (row * passes + 32), flops=4 * passes * c["N"] * c["V"])


# ------------------------------------------------------------------ the definition, in 64 bits


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] in ("w4", "embed_w4"):
        def rows(at):
            b = s["packed"][at].to(torch.int64)
            w = torch.empty(b.shape[0], c["d"], device="cuda", dtype=torch.float64)
            w[:, 0::2], w[:, 1::2] = (b % 16).double(), (b // 16).double()
            group = torch.arange(c["d"], device="cuda") // c["g"]
            w -= 8.0 if s["zeros"] is None else s["zeros"][at].double()[:, group]
            return w * s["scales"][at].double()[:, group]

        if c["op"] == "embed_w4":
            return torch.where((s["ids"] < 0)[:, None], 0.0, rows(s["ids"].clamp(min=0)) * s["scale"])
        out = torch.empty(c["B"], c["V"], device="cuda", dtype=torch.float64)
        for v in range(0, c["V"], 8192):
            out[:, v:v + 8192] = s["hidden"].double() @ rows(slice(v, v + 8192)).t()
        return out
    if c["op"] == "embed":
        return torch.where((s["ids"] < 0)[:, None], 0.0, s["table"].double()[s["ids"].clamp(min=0)] * s["scale"])
    if c["op"] == "embed_grad":
        grad = torch.zeros(c["V"] + 1, c["d"], device="cuda", dtype=torch.float64)  # the last row takes the padding
        grad.index_add_(0, torch.where(s["ids"] < 0, c["V"], s["ids"]), s["dout"].double())
        grad = grad[:-1] * s["scale"]
        return grad if s["base"] is None else grad + s["base"].double()
    T, N, V = c["temperature"], c["N"], c["V"]
    a = {k: s[k].double() for k in ("old", "adv", "ref", "weights", "lse", "dlogp") if s.get(k) is not None}
    grad = torch.empty(N, V, device="cuda", dtype=torch.float64) if c["op"] != "logp" else None
    loss, logp, lse = (torch.zeros(N, device="cuda", dtype=torch.float64) for _ in range(3))
    step = max(1, 60_000_000 // V)
    for i in range(0, N, step):
        rows = slice(i, i + step)
        x = s["logits"][rows].double() / T
        ids, ok = s["ids"][rows].clamp(min=0), s["ids"][rows] >= 0
        here = torch.arange(ids.shape[0], device="cuda")
        norm = torch.logsumexp(x, 1) if c["op"] != "logp_grad" else a["lse"][rows]
        lp = x[here, ids] - norm
        lse[rows], logp[rows] = norm, torch.where(ok, lp, 0.0)
        if c["op"] == "logp":
            continue
        if c["op"] == "logp_grad":
            d = a["dlogp"][rows]
        else:
            A, lr = a["adv"][rows], lp - a["old"][rows]
            inside = torch.where(A >= 0, lr <= math.log(1.2), lr >= math.log(0.8))
            bound = torch.where(A >= 0, 1.2, 0.8)
            value = -A * torch.where(inside, lr.exp(), bound)
            d = torch.where(inside, -A * lr.exp(), 0.0)
            if "ref" in a:
                q = (a["ref"][rows] - lp).exp()
                value = value + c["kl"] * (q - 1 - (a["ref"][rows] - lp))
                d = d + c["kl"] * (1 - q)
            loss[rows] = torch.where(ok, value, 0.0)
            d = d * a["weights"][rows]
        d = torch.where(ok, d, 0.0) / T
        p = (x - norm[:, None]).exp()
        p[here, ids] -= 1
        grad[rows] = p * -d[:, None]
    if c["op"] == "logp":
        return dict(logp=logp, lse=lse)
    return grad if c["op"] == "logp_grad" else dict(loss=loss, logp=logp, dlogits=grad)
