"""What is measured of the operators around a batch's shared projections: the residual's addition with the RMS norm
and its 8-bit codes, low-rank adapters of many requests, log-probabilities of tokens with their alternatives.
"""
import math

import torch

own = False

GROUP = 128      # columns that share an activation scale


def listed():
    return [
        # the norm before a projection of one token, as the codes that the W4A8 product reads: all launch and latency
        {"name": "norm_q8_1x4096", "op": "norm", "rows": 1, "n": 4096, "delta": True, "codes": True, "gap": 0},
        # the verify step of a draft of 8, in fp32 for INT8 weights
        {"name": "norm_9x2048", "op": "norm", "rows": 9, "n": 2048, "delta": True, "codes": False, "gap": 0},
        # a chunk of a prompt in codes, its rows cut out of wider ones
        {"name": "norm_q8_512x4096", "op": "norm", "rows": 512, "n": 4096, "delta": True, "codes": True, "gap": 2048},
        # a long prompt before its INT8 product
        {"name": "norm_4099x4096", "op": "norm", "rows": 4099, "n": 4096, "delta": True, "codes": False, "gap": 0},
        # one conversation with a small adapter
        {"name": "lora_1x2048_r8", "op": "lora", "rows": 1, "n": 2048, "m": 2048, "rank": 8, "adapters": 4, "type": "bf16", "spread": "own", "uneven": False},
        # a decode step in which every request has an adapter of its own
        {"name": "lora_32x4096_r16", "op": "lora", "rows": 32, "n": 4096, "m": 4096, "rank": 16, "adapters": 48, "type": "fp16", "spread": "own", "uneven": False},
        # a wider batch before a narrowing projection: a few adapters have most of the requests, ranks differ, some requests have none
        {"name": "lora_120x14336to4096_r64", "op": "lora", "rows": 120, "n": 14336, "m": 4096, "rank": 64, "adapters": 16, "type": "bf16", "spread": "skewed", "uneven": True},
        # packed prompts of eight requests
        {"name": "lora_4099x4096_r32", "op": "lora", "rows": 4099, "n": 4096, "m": 4096, "rank": 32, "adapters": 8, "type": "fp16", "spread": "runs", "uneven": False},
        # the token just sampled, with the five best beside it
        {"name": "logprobs_1x32000_k5", "op": "logprobs", "rows": 1, "vocab": 32000, "k": 5, "tokens": 1, "masked": False},
        # a batch over a large vocabulary, the answers of a constrained decoder: most of the vocabulary masked
        {"name": "logprobs_32x128000_k20", "op": "logprobs", "rows": 32, "vocab": 128000, "k": 20, "tokens": 1, "masked": True},
        # four choices compared at each of a few positions, no alternatives
        {"name": "logprobs_9x32000_t4", "op": "logprobs", "rows": 9, "vocab": 32000, "k": 0, "tokens": 4, "masked": False},
        # a prompt scored, rows of odd length
        {"name": "logprobs_2047x32003_k8", "op": "logprobs", "rows": 2047, "vocab": 32003, "k": 8, "tokens": 1, "masked": False},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "lora", "logprobs"])
    if op == "norm":
        n = rng.choice([2048, 4096, 5632, 14336, spread(1, 20000), 8 * spread(1, 1000)])
        rows = spread(1, max(1, min(6000, 4099 * 4096 // n)))
        return {"op": op, "rows": rows, "n": n, "delta": rng.random() < 0.7, "codes": rng.random() < 0.5, "gap": rng.choice([0, 0, 4, 1, 64])}
    if op == "lora":
        n, m = rng.choice([(2048, 2048), (4096, 4096), (4096, 14336), (14336, 4096), (4096, 1024), (spread(1, 6000), spread(1, 6000)), (8 * spread(1, 800), 8 * spread(1, 800))])
        rank = rng.choice([1, 8, 16, 32, 64, spread(1, 128)])
        rows = spread(1, max(1, min(4099, 4099 * 4096 * 3 // (n + 2 * m))))
        return {"op": op, "rows": rows, "n": n, "m": m, "rank": rank, "adapters": spread(1, 48 if rank <= 32 else 16), "type": rng.choice(["fp16", "bf16"]),
                "spread": rng.choice(["own", "skewed", "runs"]), "uneven": rng.random() < 0.4}
    vocab = rng.choice([32000, 32003, 50000, 128000, spread(1, 260000)])
    rows = spread(1, max(1, min(4096, 2047 * 32003 // vocab)))
    return {"op": op, "rows": rows, "vocab": vocab, "k": rng.choice([0, 1, 5, 20, spread(1, 32)]), "tokens": rng.choice([1, 1, 1, 0, spread(2, 8)]), "masked": rng.random() < 0.3}


def wide(g, rows, n, gap, scale):
    """[rows, n] of a wider tensor, some of its columns far larger than the others, as hidden states have them."""
    x = torch.randn(rows, n + gap, generator=g, device="cuda") * scale
    x = x * torch.exp(torch.randn(n + gap, generator=g, device="cuda") * 0.7)
    return x[:, :n]


def adapter_of_rows(case, g):
    """The adapter of each row on the host: each its own, a few for most rows and none for some, or runs of rows."""
    rows, n = case["rows"], case["adapters"]
    if case["spread"] == "own":
        return torch.randperm(max(rows, n), generator=g)[:rows] % n
    if case["spread"] == "skewed":
        return (torch.rand(rows, generator=g) ** 3 * (n + 1)).long() - 1
    return torch.sort(torch.randint(0, n, (rows,), generator=g)).values


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = {"case": case}
    if case["op"] == "norm":
        rows, n = case["rows"], case["n"]
        st["x"] = wide(g, rows, n, case["gap"], 2.0)
        st["delta"] = wide(g, rows, n, case["gap"], 0.5) if case["delta"] else None
        st["weight"] = torch.rand(n, generator=g, device="cuda") + 0.5
    elif case["op"] == "lora":
        rows, n, m, r, a = case["rows"], case["n"], case["m"], case["rank"], case["adapters"]
        host = torch.Generator()
        host.manual_seed(seed)
        dt = torch.float16 if case["type"] == "fp16" else torch.bfloat16
        st["ids"] = adapter_of_rows(case, host).to(torch.int32).cuda()
        st["ranks"] = torch.randint(1, r + 1, (a,), generator=host).to(torch.int32).cuda() if case["uneven"] else None
        st["scales"] = torch.rand(a, generator=g, device="cuda") * 2 + 0.5
        st["a"] = (torch.randn(a, r, n, generator=g, device="cuda") / math.sqrt(n)).to(dt)
        st["b"] = (torch.randn(a, m, r, generator=g, device="cuda") / math.sqrt(r)).to(dt)
        st["x"] = wide(g, rows, n, 0, 1.0)
        st["base"] = torch.randn(rows, m, generator=g, device="cuda")
    else:
        rows, v = case["rows"], case["vocab"]
        z = torch.randn(rows, v, generator=g, device="cuda") * 2.5
        if case["masked"]:
            z = torch.where(torch.rand(rows, v, generator=g, device="cuda") < 0.9, -math.inf, z)
        st["logits"] = z
        # tokens as a sampler picks them
        noise = -torch.log(-torch.log(torch.rand(rows, v, generator=g, device="cuda") * 0.999 + 5e-4))
        picked = (z + noise).argmax(-1, keepdim=True)
        other = torch.randint(0, v, (rows, max(0, case["tokens"] - 1)), generator=g, device="cuda")
        st["tokens"] = torch.cat([picked, other], 1)[:, :case["tokens"]].to(torch.int32)
    return st


def plain_norm(st):
    x, w, n = st["x"], st["weight"], st["case"]["n"]
    h = x + st["delta"] if st["delta"] is not None else x
    r = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5)
    p = h * w
    out = [h] if st["delta"] is not None else []
    if not st["case"]["codes"]:
        return out + [p * r]
    groups = (n + GROUP - 1) // GROUP
    p = torch.nn.functional.pad(p, (0, groups * GROUP - n)).unflatten(-1, (groups, GROUP))
    top = p.abs().amax(-1, keepdim=True)
    scale = top * r.unsqueeze(-1) / 127.0
    # the norm's factor cancels in a code, which is rounded from the quotient in 64 bits so that one next to a border
    # falls to its side; halves go away from zero
    part = 127.0 * p.double() / torch.where(top == 0, 1.0, top).double()
    code = (torch.sign(part) * torch.floor(part.abs() + (0.5 + 2.0 ** -40))).float()
    tiny = top * r.unsqueeze(-1) < 1e-10
    code, scale = torch.where(tiny, 0.0, code), torch.where(tiny, 1e-10, scale)
    return out + [(code * scale).flatten(-2)[:, :n], scale.squeeze(-1)]


def plain_lora(st):
    case, ids, x, a, b = st["case"], st["ids"].long(), st["x"], st["a"], st["b"]
    at = ids.clamp_min(0)
    row = torch.arange(case["rows"], device=x.device)
    few = case["rows"] <= 64
    # few rows take their adapters along, many go through all adapters in one product and pick theirs
    t = (a[at].float() * x.unsqueeze(1)).sum(-1) if few else (x @ a.flatten(0, 1).float().T).view(case["rows"], case["adapters"], case["rank"])[row, at]
    t = t * st["scales"][at].unsqueeze(1)
    held = (ids >= 0).unsqueeze(1)
    if st["ranks"] is not None:
        held = held & (torch.arange(case["rank"], device=x.device) < st["ranks"][at].unsqueeze(1))
    t = torch.where(held, t, 0.0)
    if few:
        return st["base"] + (b[at].float() * t.unsqueeze(1)).sum(-1)
    placed = torch.zeros(case["rows"], case["adapters"], case["rank"], device=x.device)
    placed[row, at] = t
    return st["base"] + placed.flatten(1) @ b.transpose(1, 2).flatten(0, 1).float()


def plain_logprobs(st):
    z, k = st["logits"], min(st["case"]["k"], st["case"]["vocab"])
    top = z.amax(-1, keepdim=True)
    d = z - torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    lse = torch.log(total)
    out = []
    if st["case"]["tokens"]:
        # a row whose mask leaves nothing gives no token any probability
        out.append(torch.where(total > 0, torch.gather(d, 1, st["tokens"].long()) - lse, -math.inf))
    mean = torch.where(e > 0, e * d, 0.0).sum(-1) / total.squeeze(1)
    out.append(torch.where(total > 0, lse - mean.unsqueeze(1), 0.0).squeeze(1))
    if st["case"]["k"]:
        value, order = torch.sort(d, dim=-1, descending=True, stable=True)
        value, order = value[:, :k], order[:, :k].to(torch.int32)
        held = value > -math.inf
        pad = (0, st["case"]["k"] - k)
        out.append(torch.nn.functional.pad(torch.where(held, order, -1), pad, value=-1))
        out.append(torch.nn.functional.pad(torch.where(held, value - lse, -math.inf), pad, value=-math.inf))
    return out


def run(st):
    case = st["case"]
    if not own:
        return {"norm": plain_norm, "lora": plain_lora, "logprobs": plain_logprobs}[case["op"]](st)
    from libinferbit_amd import ops

    if case["op"] == "norm":
        x, n = st["x"], case["n"]
        h = torch.empty(x.shape, device=x.device) if case["delta"] else None
        out = [h] if case["delta"] else []
        if not case["codes"]:
            y = torch.empty(x.shape, device=x.device)
            ops.add_rmsnorm(y, x, st["weight"], 1e-5, delta=st["delta"], h=h)
            return out + [y]
        groups = (n + GROUP - 1) // GROUP
        q, s = torch.empty(x.shape, dtype=torch.int8, device=x.device), torch.empty(x.shape[0], groups, device=x.device)
        ops.add_rmsnorm(None, x, st["weight"], 1e-5, delta=st["delta"], h=h, q=q, s=s)
        # the values that the codes stand for
        held = torch.mul(q.view(-1, groups, GROUP), s.unsqueeze(-1)).view(q.shape) if n % GROUP == 0 else torch.mul(q, s.repeat_interleave(GROUP, 1)[:, :n])
        return out + [held, s]
    if case["op"] == "lora":
        out = torch.empty_like(st["base"])
        ops.lora(out, st["x"], st["a"], st["b"], st["ids"], base=st["base"], scales=st["scales"], ranks=st["ranks"])
        return out
    z, k, rows = st["logits"], case["k"], case["rows"]
    lp = torch.empty(rows, case["tokens"], device=z.device) if case["tokens"] else None
    entropy = torch.empty(rows, device=z.device)
    ids, top = (torch.empty(rows, k, dtype=torch.int32, device=z.device), torch.empty(rows, k, device=z.device)) if k else (None, None)
    ops.logprobs(lp, z, st["tokens"] if case["tokens"] else None, entropy=entropy, top_ids=ids, top_logprobs=top)
    return [t for t in (lp, entropy, ids, top) if t is not None]


def ranks_used(case):
    """(adapters that some row takes, about: what a sampler's ids leave; their rows of rank)."""
    n = min(case["adapters"], case["rows"])
    return n * (case["rank"] / 2 if case["uneven"] else case["rank"])


def work(case):
    if case["op"] == "norm":
        size = case["rows"] * case["n"]
        out = 1 + 4 / GROUP if case["codes"] else 4
        return {"bytes": size * ((12 if case["delta"] else 4) + out) + 4 * case["n"], "flops": 6 * size}
    if case["op"] == "lora":
        rows, n, m = case["rows"], case["n"], case["m"]
        return {"bytes": 4 * rows * (n + 2 * m) + 2 * ranks_used(case) * (n + m), "flops": 2 * rows * (n + m) * (case["rank"] / 2 if case["uneven"] else case["rank"])}
    rows = case["rows"]
    return {"bytes": 4 * rows * case["vocab"] + rows * (8 * case["tokens"] + 4 + 8 * case["k"]), "flops": 6 * rows * case["vocab"]}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        # the sum and the products as they are named: h and h * weight are rounded to 32 bits, nothing else is
        h = (st["x"].double() + st["delta"].double()).float() if case["delta"] else st["x"]
        p = (h.double() * st["weight"].double()).float().double()
        root = torch.sqrt(h.double().square().sum(-1) / case["n"] + 1e-5)
        out = [h.double()] if case["delta"] else []
        if not case["codes"]:
            return out + [p / root.unsqueeze(1)]
        values, scales = torch.empty_like(p), []
        for at in range(0, case["n"], GROUP):
            part = p[:, at:at + GROUP]
            step = part.abs().amax(1, keepdim=True) / 127
            steps = torch.where(step > 0, part.abs() / step, 0.0)
            low = torch.floor(steps)
            code = (low + (steps - low >= 0.5 - 2.0 ** -40)) * torch.sign(part)
            scale = step / root.unsqueeze(1)
            small = scale * 127 < 1e-10
            values[:, at:at + GROUP] = torch.where(small, 0.0, code * scale)
            scales.append(torch.where(small, 1e-10, scale))
        return out + [values, torch.cat(scales, 1)]
    if case["op"] == "lora":
        out = st["base"].double()
        ids = st["ids"].tolist()
        for i in sorted(set(ids) - {-1}):
            r = case["rank"] if st["ranks"] is None else int(st["ranks"][i])
            rows = torch.tensor([j for j, k in enumerate(ids) if k == i], device="cuda")
            t = torch.mm(st["x"][rows].double(), st["a"][i, :r].double().T.contiguous())
            out[rows] += torch.mm(t, st["b"][i, :, :r].double().T.contiguous()) * float(st["scales"][i])
        return out
    z = st["logits"]
    parts = []
    for at in range(0, z.shape[0], 256):
        part = z[at:at + 256].double()
        lp = torch.where((part > -math.inf).any(-1, keepdim=True), torch.log_softmax(part, -1), -math.inf)
        p = torch.exp(lp)
        got = [torch.gather(lp, 1, st["tokens"][at:at + 256].long())] if case["tokens"] else []
        got.append(-torch.where(p > 0, p * lp, 0.0).sum(-1))
        if case["k"]:
            best = torch.topk(lp, min(case["k"], case["vocab"]), dim=-1).values
            got.append(torch.nn.functional.pad(best, (0, case["k"] - best.shape[1]), value=-math.inf))
        parts.append(got)
    out = [torch.cat(p) for p in zip(*parts)]
    return out[:-1] + [None] + out[-1:] if case["k"] else out
