"""Cases and plain forms of the operators that train on queries, keys and values.

Two operators, each as a user's program calls it:

* ``attend``: one training pass of SBLocal attention: the output and the gradients of query, key and value.  Row i
  weighs a key inside its window i - w/2 ... i - w/2 + w - 1 with exp(tau q.k) and any other real key with the
  low-rank estimate phi(q).phi(k), phi(x) = exp(+-sqrt(tau) W x - tau |x|^2 / 2) / sqrt(m); the weights of a row are
  divided by their sum.
* ``rotate``: root-mean-square norm of every query and key head with a learned weight, then the rotation of pairs of
  its first ``rotary`` entries by position * theta^(-2 i / rotary), forward alone or with the gradients of query,
  key and the two weights.

A case is a dict of plain values.  ``own`` chooses between the framework's kernels and the plain form below, which is
written in elementary torch operations with fp32 arithmetic (fp64 for angles).
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def attend(name, dtype, B, H, T, S, E, D, r, w, temp=0.0, ragged=False):
    return {"name": name, "op": "attend", "dtype": dtype, "B": B, "H": H, "T": T, "S": S, "E": E, "D": D, "r": r,
            "w": w, "temp": temp, "ragged": ragged}


def rotate(name, dtype, B, T, Hq, Hk, E, rotary, interleaved, positions, grad):
    return {"name": name, "op": "rotate", "dtype": dtype, "B": B, "T": T, "Hq": Hq, "Hk": Hk, "E": E, "rotary": rotary,
            "interleaved": interleaved, "positions": positions, "grad": grad}


def listed():
    return [
        # the layer's own test grid: odd sizes, more queries than keys, padded keys; a call that is all latency
        attend("attend fp32 47x39 odd", "fp32", 18, 7, 47, 39, 21, 17, 13, 28, 0.235, True),
        # first token-to-token stage of the vision model: one head, temperature from the input width
        attend("attend fp32 3136", "fp32", 8, 1, 3136, 3136, 64, 64, 128, 256, 147 ** -0.5),
        # its second stage in bf16: a sequence of about three windows, six and a bit 128-row tiles
        attend("attend bf16 784", "bf16", 8, 1, 784, 784, 64, 64, 128, 256, 576 ** -0.5),
        # a padded batch of texts of different lengths, none a multiple of a tile
        attend("attend bf16 2047 ragged", "bf16", 8, 4, 2047, 2047, 64, 64, 128, 128, 0.0, True),
        # the two sharded benchmark batches of the framework, on one device
        attend("attend bf16 4096", "bf16", 4, 12, 4096, 4096, 64, 64, 128, 256),
        attend("attend bf16 16384", "bf16", 2, 16, 16384, 16384, 64, 64, 128, 256),
        # the long-sequence heads, a quarter of that configuration's sequence
        attend("attend bf16 32768 d128", "bf16", 1, 8, 32768, 32768, 128, 128, 256, 512),
        # serving: one new token in each of eight sequences, far from the start
        rotate("rotate bf16 tokens", "bf16", 8, 1, 16, 16, 64, 64, False, True, False),
        # a prompt of odd length with fewer key heads, neighbours as pairs, part of the head rotated
        rotate("rotate fp32 1021 odd", "fp32", 3, 1021, 12, 4, 96, 40, True, True, False),
        # a padded batch in training, every gradient
        rotate("rotate bf16 2047 train", "bf16", 8, 2047, 4, 4, 64, 64, False, True, True),
        # the two benchmark head shapes in training
        rotate("rotate bf16 16384 train", "bf16", 2, 16384, 16, 16, 64, 64, False, False, True),
        rotate("rotate bf16 32768 train d128", "bf16", 1, 32768, 8, 8, 128, 128, True, False, True),
    ]


def spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.6:
        dtype, E, D, r = rng.choice([("bf16", 64, 64, 128), ("bf16", 64, 64, 128), ("bf16", 128, 128, 256),
                                     ("fp32", 64, 64, 128), ("fp32", 0, 0, 0), ("bf16", 0, 0, 0)])
        if E == 0:
            E, D, r = rng.randint(4, 128), rng.randint(4, 128), spread(rng, 4, 200)
        fast = dtype == "bf16" and (E, D, r) in ((64, 64, 128), (128, 128, 256))
        T = spread(rng, 1, 16384 if fast else 3500)
        # (with a single key the gradients of queries and keys are zero: nothing to compare)
        S = max(2, T if rng.random() < 0.7 else spread(rng, 1, 16384 if fast else 3500))
        w = spread(rng, 1, 1024)
        room = (1 << 19 if E == 64 else 1 << 18) if fast else 1 << 15
        units = max(1, min(64, room * 256 // (max(T, S) * max(256, w))))
        B = spread(rng, 1, units)
        H = spread(rng, 1, max(1, units // B))
        temp = 0.0 if rng.random() < 0.6 else rng.uniform(0.04, 0.3)
        c = attend("", dtype, B, H, T, S, E, D, r, w, temp, rng.random() < 0.5)
    else:
        E = rng.choice([64, 64, 128, 128, 2 * rng.randint(4, 128)])
        rotary = E if rng.random() < 0.5 else 2 * rng.randint(0, E // 2)
        T = spread(rng, 1, 32768)
        Hq = spread(rng, 1, 32)
        Hk = Hq if rng.random() < 0.5 else rng.randint(1, Hq)
        rows = max(1, (1 << 19) // (T * Hq))
        B = spread(rng, 1, min(rows, 64))
        c = rotate("", rng.choice(["bf16", "bf16", "fp32"]), B, T, Hq, Hk, E, rotary, rng.random() < 0.5,
                   rng.random() < 0.5, rng.random() < 0.6)
    del c["name"]
    return c


def temperature(case):
    return case["temp"] if case["temp"] > 0 else case["E"] ** -0.5


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "attend":
        B, H, T, S, E, D, r, w = (case[n] for n in ("B", "H", "T", "S", "E", "D", "r", "w"))
        m = 2 * r
        # q, k, v and the output's gradient read, the output and three gradients written; the projection
        moved = B * H * size * (2 * T * E + 2 * S * E + 2 * S * D + 2 * T * D) + 4 * r * E
        # pairs (query, key) inside a window: products q.k, dout.v (E, D), their three gradients, and the estimate's
        # own phi.phi with its two gradients (m each); forward once more q.k, phi.phi, weights.v
        pairs = T * min(w, S)
        band = pairs * ((E + m + D) + (E + D + 2 * E + D + 3 * m))
        # per row: projections and their gradients, and the products with the two m x D summaries
        rows = (T + S) * (2 * r * E + 2 * r * E) + (2 * T + S) * m * D + (T + 2 * S) * m * D
        return {"bytes": moved, "flops": 2 * B * H * (band + rows)}
    x = case["B"] * case["T"] * (case["Hq"] + case["Hk"]) * case["E"]
    # forward: read and write; gradients: inputs and output gradients read, input gradients written
    return {"bytes": x * size * (5 if case["grad"] else 2), "flops": x * (20 if case["grad"] else 8)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "attend":
        B, H, T, S, E, D, r = (case[n] for n in ("B", "H", "T", "S", "E", "D", "r"))
        # logits of unit scale, as the layer's benchmark draws them
        scale = (temperature(case) * E) ** -0.5
        blocks = -(-r // E)
        rows = torch.linalg.qr(normal(blocks, E, E))[0].transpose(1, 2).reshape(blocks * E, E)[:r]
        state = {"query": (normal(B, T, H, E) * scale).to(dtype).requires_grad_(),
                 "key": (normal(B, S, H, E) * scale).to(dtype).requires_grad_(),
                 "value": normal(B, S, H, D).to(dtype).requires_grad_(),
                 "dout": normal(B, T, H, D).to(dtype),
                 "projection": (rows * normal(r, E).norm(dim=1, keepdim=True)).contiguous(),
                 "lengths": None}
        if case["ragged"]:
            lengths = torch.randint(max(1, S // 3), S + 1, (B,), generator=g, device="cuda")
            lengths[int(seed) % B] = S
            state["lengths"] = lengths
    else:
        B, T, Hq, Hk, E = (case[n] for n in ("B", "T", "Hq", "Hk", "E"))
        state = {"query": normal(B, T, Hq, E).to(dtype), "key": normal(B, T, Hk, E).to(dtype),
                 "query_weight": 1 + 0.1 * normal(E), "key_weight": 1 + 0.1 * normal(E), "positions": None}
        if case["positions"]:
            # sequences that begin at different places of long contexts
            first = torch.randint(0, 1 << 20, (B, 1), generator=g, device="cuda")
            state["positions"] = first + torch.arange(T, device="cuda")
        if case["grad"]:
            for n in ("query", "key", "query_weight", "key_weight"):
                state[n].requires_grad_()
            state["dquery_out"], state["dkey_out"] = normal(B, T, Hq, E).to(dtype), normal(B, T, Hk, E).to(dtype)
    state["case"] = dict(case)
    return state


def run(state):
    case = state["case"]
    if own:
        return run_own(state)
    with torch.no_grad():
        if case["op"] == "attend":
            return plain_attend(state["query"], state["key"], state["value"], state["dout"], state["projection"],
                                case["w"], temperature(case), state["lengths"])
        out = {}
        for side in ("query", "key"):
            out.update(plain_rotate(side, state, case))
        return out


def run_own(state):
    from fly_b200 import ops

    case = state["case"]
    if case["op"] == "attend":
        out = ops.sblocal_attention(state["query"], state["key"], state["value"], state["projection"], case["w"],
                                    temperature(case), key_lengths=state["lengths"])
        dq, dk, dv = torch.autograd.grad(out, (state["query"], state["key"], state["value"]), state["dout"])
        return {"out": out, "dquery": dq, "dkey": dk, "dvalue": dv}
    q, k = ops.qk_norm_rotary(state["query"], state["key"], state["query_weight"], state["key_weight"],
                              positions=state["positions"], rotary_dim=case["rotary"], theta=10000.0,
                              interleaved=case["interleaved"], eps=1e-6)
    if not case["grad"]:
        return {"query": q, "key": k}
    names = ("query", "key", "query_weight", "key_weight")
    grads = torch.autograd.grad((q, k), [state[n] for n in names], (state["dquery_out"], state["dkey_out"]))
    return {"query": q, "key": k, **{"d" + n: x for n, x in zip(names, grads)}}


# ---- plain forms ------------------------------------------------------------------------------------------------


def in_blocks(x, block):
    """(B, H, N, ...) -> (B, H, blocks, block, ...), zeros behind the end."""
    n = x.shape[2]
    full = -(-n // block) * block
    if full != n:
        x = torch.cat([x, x.new_zeros(*x.shape[:2], full - n, *x.shape[3:])], dim=2)
    return x.reshape(*x.shape[:2], full // block, block, *x.shape[3:])


def plain_attend(query, key, value, dout, projection, w, tau, lengths):
    q, k, v, do = (x.permute(0, 2, 1, 3).float() for x in (query, key, value, dout))
    T, S, m = q.shape[2], k.shape[2], 2 * projection.shape[0]
    proj = math.sqrt(tau) * projection.float()
    dev = q.device
    real = torch.arange(S, device=dev)[None] < (lengths[:, None] if lengths is not None else S)  # (B or 1, S)
    real = real[:, None]
    # features, each divided by its own scale: exp(u - max) for queries, exp(u - tau |k|^2 / 2 - max) for keys
    uq, uk = q @ proj.T, k @ proj.T
    gk = 0.5 * tau * (k * k).sum(-1, keepdim=True)
    mq = uq.abs().amax(-1, keepdim=True)
    beta = (uk.abs().amax(-1, keepdim=True) - gk).amax(2, keepdim=True)
    fq = torch.exp(torch.cat([uq, -uq], -1) - mq)
    fk = torch.exp(torch.cat([uk, -uk], -1) - gk - beta) * real[..., None]
    scale = (mq - 0.5 * tau * (q * q).sum(-1, keepdim=True) + beta - math.log(m))[..., 0]
    kv, ksum = fk.transpose(2, 3) @ v, fk.sum(2)
    # windows: block b of queries sees keys from b * block - w // 2 on, block + w - 1 of them
    block = min(128, max(T, S))
    j, row = torch.arange(block + w - 1, device=dev), torch.arange(block, device=dev)
    inside = (j[None] >= row[:, None]) & (j[None] < row[:, None] + w)

    def window(n, other, low):
        start = torch.arange(-(-n // block), device=dev)[:, None] * block
        at = start + low + j
        seen = (at >= 0) & (at < other)
        return at.clamp(0, other - 1), seen, (start + row < n)[:, :, None] & inside & seen[:, None]

    at, _, see = window(T, S, -(w // 2))
    see = see & real[:, :, at][:, :, :, None]
    kw, vw, fw = k[:, :, at], v[:, :, at], fk[:, :, at]
    qb, fb, ob = in_blocks(q, block), in_blocks(fq, block), in_blocks(do, block)

    def rows(x):
        return x.reshape(*x.shape[:2], -1, *x.shape[4:])[:, :, :T]

    logit = (tau * (qb @ kw.transpose(3, 4))).masked_fill(~see, -math.inf)
    near = (fb @ fw.transpose(3, 4)) * see
    far = (fq @ ksum[..., None])[..., 0] - rows(near.sum(-1))
    norm = torch.logaddexp(rows(torch.logsumexp(logit, -1)), torch.log(far.clamp_min(1e-24)) + scale)
    share = torch.exp(scale - norm)[..., None]
    normb, shareb = in_blocks(norm, block)[..., None], in_blocks(share, block)
    p = torch.exp(logit - normb)
    out = rows((p - near * shareb) @ vw) + share * (fq @ kv)
    delta = (do * out).sum(-1, keepdim=True)
    pull = (ob @ vw.transpose(3, 4) - in_blocks(delta, block)) * see
    dq = tau * rows((p * pull) @ kw)
    dfq = fq * share * (do @ kv.transpose(2, 3) - delta * ksum[:, :, None] - rows(pull @ fw))
    r = m // 2
    dq = dq + (dfq[..., :r] - dfq[..., r:]) @ proj - tau * q * dfq.sum(-1, keepdim=True)
    del kw, vw, fw, logit, near, p, pull
    # the same from the keys' side: block b of keys is seen by queries from b * block + w // 2 - w + 1 on
    psi = fq * share
    summary, lost = psi.transpose(2, 3) @ do, (psi * delta).sum(2)
    at, _, see = window(S, T, w // 2 - w + 1)
    see = see & in_blocks(real.expand(-1, 1, S), block)[..., None]
    qw, ow, fw, nw, tw = q[:, :, at], do[:, :, at], psi[:, :, at], norm[:, :, at], delta[:, :, at]
    kb, vb, fb = in_blocks(k, block), in_blocks(v, block), in_blocks(fk, block)

    def keys(x):
        return x.reshape(*x.shape[:2], -1, *x.shape[4:])[:, :, :S]

    p = torch.exp((tau * (kb @ qw.transpose(3, 4)) - nw[:, :, :, None]).masked_fill(~see, -math.inf))
    near = (fb @ fw.transpose(3, 4)) * see
    pull = (vb @ ow.transpose(3, 4) - tw.transpose(3, 4)) * see
    dv = keys((p - near) @ ow) + fk @ summary
    dfk = fk * (v @ summary.transpose(2, 3) - lost[:, :, None] - keys(pull @ fw))
    dk = tau * keys((p * pull) @ qw) + (dfk[..., :r] - dfk[..., r:]) @ proj - tau * k * dfk.sum(-1, keepdim=True)
    back = lambda x, like: x.permute(0, 2, 1, 3).to(like.dtype)  # noqa: E731
    return {"out": back(out, query), "dquery": back(dq, query), "dkey": back(dk, key), "dvalue": back(dv, value)}


def angles(state, case, dtype):
    rotary = case["rotary"]
    pos = state["positions"]
    if pos is None:
        pos = torch.arange(case["T"], device=state["query"].device)[None]
    rate = 10000.0 ** (-torch.arange(0, rotary, 2, device=pos.device, dtype=torch.float64) / max(rotary, 1))
    a = pos.double()[..., None, None] * rate          # (B or 1, T, 1, rotary / 2)
    return torch.cos(a).to(dtype), torch.sin(a).to(dtype)


def pairs(x, case):
    """The two entries of each rotated pair, and the entries behind them."""
    half = case["rotary"] // 2
    if case["interleaved"]:
        return x[..., 0:2 * half:2], x[..., 1:2 * half:2], x[..., 2 * half:]
    return x[..., :half], x[..., half:2 * half], x[..., 2 * half:]


def unpair(a, b, rest, case):
    if case["interleaved"]:
        return torch.cat([torch.stack([a, b], -1).flatten(-2), rest], -1)
    return torch.cat([a, b, rest], -1)


def plain_rotate(side, state, case):
    x, weight = state[side].float(), state[side + "_weight"].float()
    cos, sin = angles(state, case, torch.float32)
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    unit = x * rstd
    a, b, rest = pairs(unit * weight, case)
    out = {side: unpair(a * cos - b * sin, b * cos + a * sin, rest, case).to(state[side].dtype)}
    if case["grad"]:
        a, b, rest = pairs(state["d" + side + "_out"].float(), case)
        dz = unpair(a * cos + b * sin, b * cos - a * sin, rest, case)
        dunit = dz * weight
        out["d" + side] = (rstd * (dunit - unit * (dunit * unit).mean(-1, keepdim=True))).to(state[side].dtype)
        out["d" + side + "_weight"] = (dz * unit).sum((0, 1, 2)).to(state[side + "_weight"].dtype)
    return out


# ---- the definition in 64 bits ----------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attend":
        with torch.no_grad():
            return exact_attend(state, case)
    return exact_rotate(state, case)


def exact_attend(state, case):
    """Every weight of every row, (query rows) x (all keys) at a time."""
    tau, w, S, T = temperature(case), case["w"], case["S"], case["T"]
    W = state["projection"].double()
    m = 2 * W.shape[0]
    grads = {n: torch.zeros(state[n].shape, dtype=torch.float64, device="cuda")
             for n in ("query", "key", "value", "dout")}
    step = max(1, (1 << 27) // S)
    at = torch.arange(S, device="cuda")

    def features(x):
        u = math.sqrt(tau) * (x @ W.T)
        return torch.exp(torch.cat([u, -u], 1) - tau * (x * x).sum(1, keepdim=True) / 2 - math.log(m) / 2)

    def through(x, f, df):
        """Gradient of x where f = features(x) has the gradient df."""
        a = f * df
        return math.sqrt(tau) * (a[:, :m // 2] - a[:, m // 2:]) @ W - tau * x * a.sum(1, keepdim=True)

    for b in range(case["B"]):
        n = S if state["lengths"] is None else int(state["lengths"][b])
        for h in range(case["H"]):
            q, k, v, do = (state[x][b, :, h].double() for x in ("query", "key", "value", "dout"))
            fk = features(k)
            dfk = torch.zeros_like(fk)
            for i in range(0, T, step):
                x, o = q[i:i + step], do[i:i + step]
                row = torch.arange(i, i + x.shape[0], device="cuda")[:, None]
                near = (at >= row - w // 2) & (at < row - w // 2 + w) & (at < n)
                away = ~near & (at < n)
                fx = features(x)
                weight = torch.where(near, torch.exp(tau * x @ k.T), fx @ fk.T).masked_fill_(~(near | away), 0)
                total = weight.sum(1, keepdim=True).clamp_min(1e-300)
                weight /= total
                y = weight @ v
                grads["dout"][b, i:i + step, h] = y
                grads["value"][b, :, h] += weight.T @ o
                g = o @ v.T - (o * y).sum(1, keepdim=True)
                s = (weight * g).masked_fill_(~near, 0)
                g = (g / total).masked_fill_(~away, 0)
                grads["query"][b, i:i + step, h] = tau * s @ k + through(x, fx, g @ fk)
                grads["key"][b, :, h] += tau * s.T @ x
                dfk += g.T @ fx
            grads["key"][b, :, h] += through(k, fk, dfk)
    return {"out": grads["dout"], "dquery": grads["query"], "dkey": grads["key"], "dvalue": grads["value"]}


def exact_rotate(state, case):
    """Pairs as complex numbers, gradients by differentiating the definition."""
    half = case["rotary"] // 2
    order = torch.arange(case["E"], device="cuda")
    if half and not case["interleaved"]:
        order[:2 * half] = torch.arange(2 * half, device="cuda").reshape(2, half).T.reshape(-1)
    pos = state["positions"] if state["positions"] is not None else torch.arange(case["T"], device="cuda")[None]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       pos.double()[..., None, None]
                       * torch.exp(torch.arange(half, device="cuda").double() * (-2 * math.log(10000.0) / max(2 * half, 1))))
    out = {}
    for side in ("query", "key"):
        x = state[side].detach().double().requires_grad_()
        weight = state[side + "_weight"].detach().double().requires_grad_()
        z = (x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight)[..., order]
        pair = torch.view_as_complex(z[..., :2 * half].reshape(*z.shape[:-1], half, 2).contiguous()) * turn
        y = torch.cat([torch.view_as_real(pair).flatten(-2), z[..., 2 * half:]], -1)[..., torch.argsort(order)]
        out[side] = y.detach()
        if case["grad"]:
            dx, dw = torch.autograd.grad(y, (x, weight), state["d" + side + "_out"].double())
            out["d" + side], out["d" + side + "_weight"] = dx, dw
    return out
