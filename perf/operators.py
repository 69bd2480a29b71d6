"""Timing cases of the operators on sparse rows of scores: routing, the gradient of stored values, distillation.

Every case names one family, i.e. one entry point and the direction in which a program calls it:

    route        ``ops.route``: scores of tokens for experts in, the CSR matrix tokens x experts out (inference)
    route_train  the same and the gradient of the scores
    values       ``ops.sddmm``: the gradient of a product for the matrix's stored values
    product      ``ops.weighted_spmm`` and its gradients for the values and for B (a training step)
    distill      ``ops.distill_loss``: a teacher's entries against a student's logits (evaluation)
    distill_train  the same and the gradient of the logits
    distill_step ``ops.distill_loss_grad``: loss and gradient in one pass

Inputs are made on the GPU from the seed alone.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _route(family, T, E, k, dtype, **more):
    base = dict(family=family, T=T, E=E, k=k, dtype=dtype, score="softmax", bias=False, groups=1, top_groups=1, group_top=1,
                renormalize=True, scale=1.0, masked=0.0)
    return {**base, **more}


def _matrix(family, M, Kd, Nd, mean, kind):
    return dict(family=family, M=M, Kd=Kd, Nd=Nd, mean=float(mean), kind=kind)


def _distill(family, T, V, k, dtype, **more):
    return {**dict(family=family, T=T, V=V, k=k, dtype=dtype, ragged=False, temperature=1.0, log_probs=False), **more}


def listed():
    return [
        # one step of eight sequences: nothing but latency
        dict(_route("route", 8, 128, 4, "bf16"), name="route_decode"),
        # a long prompt through a router with a balancing bias that is limited to four of eight groups
        dict(_route("route", 16384, 256, 8, "bf16", score="sigmoid", bias=True, groups=8, top_groups=4, group_top=2, scale=2.5), name="route_prompt"),
        # nothing a multiple of anything, weights as they are, some experts out of service
        dict(_route("route_train", 3001, 60, 6, "fp16", renormalize=False, masked=0.05), name="route_train_ragged"),
        # a training batch of fp32 scores
        dict(_route("route_train", 32768, 128, 8, "fp32"), name="route_train_large"),
        # the values' gradient for a handful of tokens
        dict(_matrix("values", 64, 256, 1024, 4, "slots"), name="values_small"),
        # on a graph of the size that the training case of the library's products has
        dict(_matrix("values", 1 << 18, 1 << 18, 128, 16, "zipf"), name="values_graph"),
        # rectangular, 50 columns
        dict(_matrix("values", 100003, 77777, 50, 11, "zipf"), name="values_ragged"),
        # experts' answers combined by the routing matrix, forward and both gradients
        dict(_matrix("product", 4096, 32768, 2048, 8, "slots"), name="combine_train"),
        # a few rows of a small vocabulary
        dict(_distill("distill_train", 32, 4096, 8, "bf16"), name="distill_small"),
        # odd vocabulary, rows of no entry to a hundred, softened, teacher's log-probabilities
        dict(_distill("distill_train", 1021, 50021, 100, "fp16", ragged=True, temperature=2.0, log_probs=True), name="distill_ragged"),
        # few long rows, the loss alone
        dict(_distill("distill", 4, 262144, 256, "fp32"), name="distill_long_rows"),
        # a training batch over a large vocabulary
        dict(_distill("distill_step", 4096, 131072, 64, "bf16"), name="distill_step_large"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_route(rng):
    E = _log(rng, 8, 512)
    if rng.random() < 0.5:
        E = max(8, E // 8 * 8)
    groups = rng.choice([g for g in (1, 1, 2, 4, 8) if E % g == 0 and E // g >= 2])
    top_groups = rng.randint(1, groups)
    k = min(_log(rng, 1, 16), top_groups * (E // groups))
    T = min(_log(rng, 1, 65536), 8_000_000 // E)
    return _route(rng.choice(["route", "route_train"]), T, E, k, rng.choice(sorted(TYPES)), score=rng.choice(["softmax", "sigmoid"]),
                  bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, group_top=rng.choice([1, 2]),
                  renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), masked=rng.choice([0.0, 0.0, 0.05]))


def _draw_matrix(rng):
    family = rng.choice(["values", "product"])
    kind = rng.choice(["slots", "zipf", "even"])
    if kind == "slots":
        k = rng.choice([1, 2, 4, 6, 8])
        Nd = _log(rng, 64, 4096)
        M = max(1, min(_log(rng, 1, 16384), 67_000_000 // (Nd * k)))
        return _matrix(family, M, M * k, Nd, k, kind)
    Nd = _log(rng, 8, 512)
    mean = round(math.exp(rng.uniform(math.log(2), math.log(40))), 2)
    M = max(64, min(_log(rng, 512, 1 << 19), int(4e8 / (Nd * mean))))
    return _matrix(family, M, M if rng.random() < 0.4 else _log(rng, 512, 1 << 19), Nd, mean, kind)


def _draw_distill(rng):
    V = _log(rng, 1000, 262144)
    T = max(1, min(_log(rng, 1, 16384), 300_000_000 // V))
    return _distill(rng.choice(["distill", "distill_train", "distill_step"]), T, V, _log(rng, 1, 256), rng.choice(sorted(TYPES)),
                    ragged=rng.random() < 0.4, temperature=rng.choice([1.0, 1.0, 2.0]), log_probs=rng.random() < 0.3)


def draw(rng):
    return rng.choice([_draw_route, _draw_matrix, _draw_distill])(rng)


# ---- inputs -----------------------------------------------------------------------------------------

def _offsets(lens):
    row_ptr = torch.zeros(lens.numel() + 1, dtype=torch.int32, device="cuda")
    row_ptr[1:] = lens.cumsum(0)
    return row_ptr


def _prepare_route(case, gen):
    T, E = case["T"], case["E"]
    x = 2.0 * torch.randn((T, E), generator=gen, device="cuda") + torch.randn((1, E), generator=gen, device="cuda")
    if case["masked"]:
        x[:, torch.rand(E, generator=gen, device="cuda") < case["masked"]] = -math.inf
    bias = 0.1 * torch.randn(E, generator=gen, device="cuda") if case["bias"] else None
    g = torch.randn(T * case["k"], generator=gen, device="cuda")
    x = x.to(TYPES[case["dtype"]])
    return dict(x=x.requires_grad_(case["family"] == "route_train"), bias=bias, g=g)


def _prepare_matrix(case, gen):
    M, Kd, Nd, mean = case["M"], case["Kd"], case["Nd"], case["mean"]
    if case["kind"] == "slots":  # each column named once: the experts' rows in the order that the routing gave them
        k = int(mean)
        cols = torch.randperm(Kd, generator=gen, device="cuda").view(M, k).sort(1).values.flatten()
        lens = torch.full((M,), k, device="cuda")
    else:
        u = torch.rand(M, generator=gen, device="cuda").double()
        # a tail of exponent 2, cut where rows hold a thousand times the shortest; or between nothing and twice the mean
        length = (1.0 / u.clamp_min(1e-9)).clamp_max(1000.0) if case["kind"] == "zipf" else u
        ends = (length.cumsum(0) * (round(M * mean) / length.sum())).round().long()
        lens = torch.diff(ends, prepend=ends.new_zeros(1))
        rows = torch.repeat_interleave(torch.arange(M, device="cuda"), lens)
        key = rows * Kd + torch.randint(0, Kd, rows.shape, generator=gen, device="cuda")
        cols = key.sort().values - rows * Kd
    B = torch.randn((Kd, Nd), generator=gen, device="cuda")
    G = torch.randn((M, Nd), generator=gen, device="cuda")
    values = torch.rand(cols.shape, generator=gen, device="cuda")
    train = case["family"] == "product"
    return dict(rp=_offsets(lens), ci=cols.to(torch.int32), va=values.requires_grad_(train), B=B.requires_grad_(train), G=G)


def _prepare_distill(case, gen):
    T, V, k = case["T"], case["V"], min(case["k"], case["V"])
    lens = torch.full((T,), k, device="cuda")
    if case["ragged"]:
        lens = torch.randint(0, k + 1, (T,), generator=gen, device="cuda")
    width = V // k
    cols = torch.arange(k, device="cuda") * width + torch.randint(0, width, (T, k), generator=gen, device="cuda")
    order = torch.rand((T, k), generator=gen, device="cuda").argsort(1)
    cols = cols.gather(1, order)  # distinct, in no order
    v = (12.0 + 2.5 * torch.randn((T, k), generator=gen, device="cuda")).sort(1, descending=True).values
    x = 2.0 * torch.randn((T, V), generator=gen, device="cuda")
    x.scatter_add_(1, cols, 0.8 * v)  # a student that has learnt most of it
    kept = torch.arange(k, device="cuda") < lens[:, None]
    if case["log_probs"]:  # what the entries left out hold is missing from the sum
        t = case["temperature"]
        mass = 0.8 + 0.2 * torch.rand((T, 1), generator=gen, device="cuda")
        v = (v / t - torch.logsumexp(v / t, 1, keepdim=True)) + mass.log()
    g = torch.rand(T, generator=gen, device="cuda") * (2.0 / T)
    if case["dtype"] == "fp16":  # a loss scaled so that its gradients do not vanish, as half precision is trained
        g = g * 1024.0
    x = x.to(TYPES[case["dtype"]])
    return dict(x=x.requires_grad_(case["family"] == "distill_train"), rp=_offsets(lens), ci=cols[kept].to(torch.int32), va=v[kept], g=g)


def _kind(case):
    return "route" if case["family"].startswith("route") else "distill" if case["family"].startswith("distill") else "matrix"


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    make = {"route": _prepare_route, "matrix": _prepare_matrix, "distill": _prepare_distill}[_kind(case)]
    return dict(make(case, gen), case=case)


# ---- plain forms ------------------------------------------------------------------------------------

def _chosen(x, case, bias):
    """Columns of the k experts of each row, ascending; scores and sums of them in 64 bits, where two may be very near."""
    T, E, G = case["T"], case["E"], case["groups"]
    d = x.double()
    if case["score"] == "sigmoid":
        c = 1.0 / (1.0 + torch.exp(-d))
    else:
        e = torch.exp(d - d.amax(1, keepdim=True))
        c = e / e.sum(1, keepdim=True)
    if bias is not None:
        c = c + bias.double()
    c = torch.where(x == -math.inf, -math.inf, c)
    if case["top_groups"] < G:
        best = c.view(T, G, E // G).sort(2, descending=True).values[:, :, :case["group_top"]].sum(2)
        order = best.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros((T, G), dtype=torch.bool, device=x.device).scatter_(1, order, True)
        left_out = ~kept.repeat_interleave(E // G, 1)
        key = torch.where(left_out, 1, 0)  # behind all others, those that are not available too
        first = c.sort(dim=1, descending=True, stable=True).indices
        second = key.gather(1, first).sort(dim=1, stable=True).indices
        return first.gather(1, second)[:, :case["k"]].sort(1).values
    return c.sort(dim=1, descending=True, stable=True).indices[:, :case["k"]].sort(1).values


def _plain_route(s):
    case = s["case"]
    T, k, scale = case["T"], case["k"], case["scale"]
    x = s["x"].detach()
    cols = _chosen(x, case, s["bias"])
    z = x.float()
    if case["score"] == "sigmoid":
        p = 1.0 / (1.0 + torch.exp(-z))
    else:
        e = torch.exp(z - z.amax(1, keepdim=True))
        p = e / e.sum(1, keepdim=True)
    chosen = p.gather(1, cols)
    total = chosen.sum(1, keepdim=True)
    share = chosen / torch.where(total > 0, total, 1.0) if case["renormalize"] else chosen
    row_ptr = torch.arange(T + 1, dtype=torch.int32, device=x.device) * k
    out = {"row_ptr": row_ptr, "col_idx": cols.flatten().to(torch.int32), "values": (share * scale).flatten()}
    if case["family"] == "route":
        return out
    g = s["g"].view(T, k)
    if case["renormalize"]:
        at = share * scale * (g - (share * g).sum(1, keepdim=True))
        at = at * (1.0 - chosen) if case["score"] == "sigmoid" else at
        dx = torch.zeros_like(z).scatter_(1, cols, at)
    elif case["score"] == "sigmoid":
        dx = torch.zeros_like(z).scatter_(1, cols, scale * chosen * (1.0 - chosen) * g)
    else:
        dense = torch.zeros_like(z).scatter_(1, cols, g)
        dx = scale * p * (dense - (chosen * g).sum(1, keepdim=True))
    return dict(out, dlogits=dx.to(x.dtype))


def _rows_of(rp, n):
    return torch.repeat_interleave(torch.arange(rp.numel() - 1, device=rp.device), (rp[1:] - rp[:-1]).long(), output_size=n)


def _plain_matrix(s):
    ci, B, G = s["ci"].long(), s["B"].detach(), s["G"]
    rows = _rows_of(s["rp"], ci.numel())
    dv = (G[rows] * B[ci]).sum(1)
    if s["case"]["family"] == "values":
        return dv
    va = s["va"].detach()[:, None]
    C = torch.zeros_like(G).index_add_(0, rows, va * B[ci])
    dB = torch.zeros_like(B).index_add_(0, ci, va * G[rows])
    return {"C": C, "dvalues": dv, "dB": dB}


def _plain_distill(s):
    case = s["case"]
    t, x = case["temperature"], s["x"].detach()
    T, V = x.shape
    ci = s["ci"].long()
    rows = _rows_of(s["rp"], ci.numel())
    z = x.float() / t
    m = z.amax(1, keepdim=True)
    lse = m[:, 0] + torch.log(torch.exp(z - m).sum(1))
    if case["log_probs"]:
        p = torch.exp(s["va"])
    else:
        v = s["va"] / t
        top = torch.full((T,), -math.inf, device=x.device).scatter_reduce_(0, rows, v, "amax")
        e = torch.exp(v - top[rows])
        p = e / torch.zeros(T, device=x.device).index_add_(0, rows, e)[rows]
    terms = torch.where(p > 0, p * (torch.log(p) - z[rows, ci] + lse[rows]), 0.0)
    loss = t * t * torch.zeros(T, device=x.device).index_add_(0, rows, terms)
    if case["family"] == "distill":
        return loss
    mass = torch.zeros(T, device=x.device).index_add_(0, rows, p)
    d = torch.exp(z - lse[:, None]).mul_(mass[:, None])
    d.view(-1).index_add_(0, rows * V + ci, -p)
    return {"loss": loss, "dlogits": d.mul_(t * s["g"][:, None]).to(x.dtype)}


# ---- one pass ---------------------------------------------------------------------------------------

def _own(s):
    from csrspmm_b200 import ops
    case = s["case"]
    family = case["family"]
    if _kind(case) == "route":
        rp, ci, va = ops.route(s["x"], case["k"], bias=s["bias"], score=case["score"], groups=case["groups"], top_groups=case["top_groups"],
                               group_top=case["group_top"], renormalize=case["renormalize"], scale=case["scale"])
        out = {"row_ptr": rp, "col_idx": ci, "values": va}
        if family == "route":
            return out
        (dx,) = torch.autograd.grad(va, s["x"], s["g"])
        return dict(out, values=va.detach(), dlogits=dx)
    if family == "values":
        return ops.sddmm(s["rp"], s["ci"], s["G"], s["B"])
    if family == "product":
        C = ops.weighted_spmm(s["rp"], s["ci"], s["va"], s["B"])
        dv, dB = torch.autograd.grad(C, (s["va"], s["B"]), s["G"])
        return {"C": C.detach(), "dvalues": dv, "dB": dB}
    how = dict(temperature=case["temperature"], log_probs=case["log_probs"])
    if family == "distill_step":
        loss, dx = ops.distill_loss_grad(s["x"], s["rp"], s["ci"], s["va"], s["g"], **how)
        return {"loss": loss, "dlogits": dx}
    loss = ops.distill_loss(s["x"], s["rp"], s["ci"], s["va"], **how)
    if family == "distill":
        return loss
    (dx,) = torch.autograd.grad(loss, s["x"], s["g"])
    return {"loss": loss.detach(), "dlogits": dx}


def run(s):
    if own:
        return _own(s)
    return {"route": _plain_route, "matrix": _plain_matrix, "distill": _plain_distill}[_kind(s["case"])](s)


# ---- the definitions in 64 bits -----------------------------------------------------------------------

def _exact_route(s, case):
    T, E, k, G = case["T"], case["E"], case["k"], case["groups"]
    x = s["x"].detach().double()
    score = torch.sigmoid(x) if case["score"] == "sigmoid" else torch.softmax(x, 1)
    choice = (score if s["bias"] is None else score + s["bias"].double()).masked_fill(x == -math.inf, -math.inf)
    # the rank of each expert: how many come before it
    if case["top_groups"] < G:
        per = choice.view(T, G, E // G)
        total = torch.topk(per, case["group_top"], 2).values.sum(2)
        number = torch.arange(G, device=x.device)
        ahead = (total[:, None, :] > total[:, :, None]) | ((total[:, None, :] == total[:, :, None]) & (number < number[:, None]))
        inside = (ahead.sum(2) < case["top_groups"])[:, :, None].expand(T, G, E // G).reshape(T, E)
    else:
        inside = torch.ones_like(choice, dtype=torch.bool)
    number = torch.arange(E, device=x.device)
    cols = torch.empty((T, k), dtype=torch.long, device=x.device)
    step = max(1, 100_000_000 // (E * E))
    for r in range(0, T, step):
        c, i = choice[r:r + step], inside[r:r + step]
        ahead = i[:, None, :] & ((c[:, None, :] > c[:, :, None]) | ((c[:, None, :] == c[:, :, None]) & (number < number[:, None])))
        cols[r:r + step] = (i & (ahead.sum(2) < k)).nonzero()[:, 1].view(-1, k)
    leaf = x.requires_grad_(True)
    weight = (torch.sigmoid(leaf) if case["score"] == "sigmoid" else torch.softmax(leaf, 1)).gather(1, cols)
    if case["renormalize"]:
        total = weight.sum(1, keepdim=True)
        weight = weight / total.masked_fill(total == 0, 1.0)
    weight = (case["scale"] * weight).flatten()
    out = {"row_ptr": torch.arange(0, T * k + 1, k, dtype=torch.int32, device=x.device), "col_idx": cols.flatten().int(), "values": weight.detach()}
    if case["family"] == "route":
        return out
    return dict(out, dlogits=torch.autograd.grad(weight, leaf, s["g"].double())[0])


def _exact_matrix(s, case):
    ci, B, G = s["ci"].long(), s["B"].detach().double(), s["G"].double()
    rows = torch.searchsorted(s["rp"].long(), torch.arange(ci.numel(), device=ci.device), right=True) - 1
    step = max(1, 200_000_000 // case["Nd"])
    dv = torch.cat([torch.einsum("en,en->e", G[rows[e:e + step]], B[ci[e:e + step]]) for e in range(0, ci.numel(), step)])
    if case["family"] == "values":
        return dv
    va = s["va"].detach().double()
    C, dB = torch.zeros_like(G), torch.zeros_like(B)
    for e in range(0, ci.numel(), step):
        r, c, w = rows[e:e + step], ci[e:e + step], va[e:e + step, None]
        C.index_add_(0, r, w * B[c])
        dB.index_add_(0, c, w * G[r])
    return {"C": C, "dvalues": dv, "dB": dB}


def _exact_distill(s, case):
    t, x = case["temperature"], s["x"].detach()
    T, V = x.shape
    loss = torch.zeros(T, dtype=torch.double, device=x.device)
    dx = None if case["family"] == "distill" else torch.empty((T, V), dtype=torch.double, device=x.device)
    kmax = max(1, case["k"])
    at = s["rp"].long()
    step = max(1, 200_000_000 // V)
    for r in range(0, T, step):
        b, e = at[r:r + step + 1][:-1, None], at[r + 1:r + step + 1][:, None]
        slot = b + torch.arange(kmax, device=x.device)
        there = slot < e
        slot = slot.clamp_max(max(0, s["ci"].numel() - 1))
        if s["ci"].numel():
            c, v = s["ci"].long()[slot].masked_fill(~there, 0), s["va"].double()[slot].masked_fill(~there, -math.inf)
        else:
            c, v = torch.zeros_like(slot), torch.full(slot.shape, -math.inf, dtype=torch.double, device=x.device)
        p = v.exp() if case["log_probs"] else torch.softmax(v / t, 1).nan_to_num(0.0)
        logq = torch.log_softmax(x[r:r + step].double() / t, 1)
        loss[r:r + step] = t * t * (torch.xlogy(p, p) - torch.where(p > 0, p * logq.gather(1, c), 0.0)).sum(1)
        if dx is not None:
            d = logq.exp() * p.sum(1, keepdim=True)
            dx[r:r + step] = d.scatter_add(1, c, -p) * (t * s["g"][r:r + step, None].double())
    return loss if dx is None else {"loss": loss, "dlogits": dx}


def exact(case, seed):
    exact_of = {"route": _exact_route, "matrix": _exact_matrix, "distill": _exact_distill}[_kind(case)]
    return exact_of(prepare(case, seed), case)


# ---- what a pass cannot do without -------------------------------------------------------------------

def work(case):
    family = case["family"]
    if _kind(case) == "route":
        T, E, k, size = case["T"], case["E"], case["k"], SIZES[case["dtype"]]
        n_bytes = T * E * size + 8.0 * T * k + 4.0 * (T + 1) + (4.0 * E if case["bias"] else 0.0)
        flops = 4.0 * T * E
        if family == "route_train":
            n_bytes += T * E * size + 4.0 * T * k
            flops += 4.0 * T * k
        return {"bytes": n_bytes, "flops": flops}
    if _kind(case) == "distill":
        T, V, size = case["T"], case["V"], SIZES[case["dtype"]]
        entries = T * case["k"] * (0.5 if case["ragged"] else 1.0)
        n_bytes = T * V * size + 8.0 * entries + 4.0 * (T + 1) + 4.0 * T
        flops = 4.0 * T * V
        if family != "distill":
            n_bytes += T * V * size + 4.0 * T
            flops += 3.0 * T * V
        return {"bytes": n_bytes, "flops": flops}
    M, Kd, Nd = case["M"], case["Kd"], case["Nd"]
    nnz = M * case["mean"]
    touched = float(Kd) if case["kind"] == "slots" else Kd * (1.0 - math.exp(-nnz / Kd))
    n_bytes = 8.0 * nnz + 4.0 * (M + 1) + 4.0 * Nd * (M + touched)
    flops = 2.0 * nnz * Nd
    if family == "product":  # C and dB out, the values in
        n_bytes += 4.0 * nnz + 4.0 * Nd * (M + Kd)
        flops *= 3
    return {"bytes": n_bytes, "flops": flops}
