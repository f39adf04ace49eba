"""The feed-forward half of a layer on quantised weights with jitnn_amd: the router of a mixture of experts (which experts a token goes
to, with which weights), the whole layer of experts, and a dense linear with bias, activation and residual in its epilogue.

`own` False: the operators' plain form in elementary torch operations.  `own` True: the calls of the package.
"""
import math

import torch

own = False

BLOCK = {"Q8_0": (8, 32, 34), "Q4_0": (2, 32, 18), "Q4_1": (3, 32, 20), "Q4_K": (12, 256, 144), "Q5_K": (13, 256, 176), "Q6_K": (14, 256, 210)}


def listed():
    return [
        # one token through the router of a layer with eight experts: the smallest call
        dict(name="route_1x8", kind="route", tokens=1, experts=8, used=2, d=4096, gating="softmax", normalise=True, scale=1.0, bias=False),
        # a prompt through the router of a layer with many small experts, sigmoid gating with a bias that balances the experts' load
        dict(name="route_1000x128_sigmoid", kind="route", tokens=1000, experts=128, used=8, d=2048, gating="sigmoid", normalise=True, scale=2.5, bias=True),
        # one token of a decode step, two of eight large experts
        dict(name="moe_1_of_8x14336", kind="moe", tokens=1, experts=8, used=2, d=4096, ffn=14336, up="Q4_K", down="Q6_K", gating="softmax", normalise=True,
             scale=1.0, bias=False, residual=True, activation="silu"),
        # one token, eight of 128 small experts: latency counts
        dict(name="moe_1_of_128x768", kind="moe", tokens=1, experts=128, used=8, d=2048, ffn=768, up="Q4_K", down="Q6_K", gating="softmax", normalise=True,
             scale=1.0, bias=False, residual=True, activation="silu"),
        # five sequences decoded together, six of 64 experts whose rows are no whole 256-value columns
        dict(name="moe_5_of_64x1408_q8_0", kind="moe", tokens=5, experts=64, used=6, d=2048, ffn=1408, up="Q8_0", down="Q8_0", gating="sigmoid", normalise=True,
             scale=2.5, bias=True, residual=True, activation="silu"),
        # a batch of 32 sequences decoded together, many small experts
        dict(name="moe_32_of_128x768", kind="moe", tokens=32, experts=128, used=8, d=2048, ffn=768, up="Q4_K", down="Q6_K", gating="softmax", normalise=True,
             scale=1.0, bias=False, residual=True, activation="silu"),
        # a batch of 24, eight large experts, five-bit weights, GELU gates
        dict(name="moe_24_of_8x14336_q5_k", kind="moe", tokens=24, experts=8, used=2, d=4096, ffn=14336, up="Q5_K", down="Q5_K", gating="softmax", normalise=True,
             scale=1.0, bias=False, residual=True, activation="gelu"),
        # a prompt of 512 tokens: the largest
        dict(name="moe_512_of_8x14336", kind="moe", tokens=512, experts=8, used=2, d=4096, ffn=14336, up="Q4_K", down="Q6_K", gating="softmax", normalise=True,
             scale=1.0, bias=False, residual=True, activation="silu"),
        # one token through a square projection: the smallest linear
        dict(name="linear_1_q8_0_4096x4096", kind="linear", fmt="Q8_0", n=4096, k=4096, rows=1, bias=True, activation="gelu", residual=True),
        # eight sequences through an up-projection with a bias and SiLU
        dict(name="linear_8_q4_k_14336x4096", kind="linear", fmt="Q4_K", n=14336, k=4096, rows=8, bias=True, activation="silu", residual=False),
        # a short prompt through a down-projection, a ragged number of rows, with bias and residual
        dict(name="linear_37_q6_k_4096x14336", kind="linear", fmt="Q6_K", n=4096, k=14336, rows=37, bias=True, activation=None, residual=True),
        # a batch of 64, rows that are no whole columns
        dict(name="linear_64_q4_0_8000x5088", kind="linear", fmt="Q4_0", n=8000, k=5088, rows=64, bias=True, activation="relu", residual=True),
    ]


LARGEST = dict(kind="moe", tokens=512, experts=8, used=2, d=4096, ffn=14336, up="Q4_K", down="Q6_K", gating="softmax", bias=False, residual=True)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _length(rng, fmt, lo, hi):
    """A row of whole blocks: 256 values, or any number of 32 where the format's blocks hold those."""
    qk = 256 if BLOCK[fmt][1] == 256 or rng.random() < 0.6 else 32
    return max(1, _log(rng, lo, hi) // qk) * qk


def draw(rng):
    kind = rng.choices(("route", "moe", "linear"), (1, 5, 3))[0]
    if kind == "linear":
        fmt = rng.choice(sorted(BLOCK))
        k = _length(rng, fmt, 512, 14336)
        n = min(_log(rng, 256, 20000), 14336 * 4096 // k)
        return dict(kind=kind, fmt=fmt, n=n, k=k, rows=rng.choice((1, rng.randint(2, 8), rng.randint(9, 64))), bias=rng.random() < 0.6,
                    activation=rng.choice((None, "relu", "silu", "gelu", "gelu_tanh")), residual=rng.random() < 0.6)
    experts = _log(rng, 4, 256)
    case = dict(kind=kind, tokens=0, experts=experts, used=min(experts, rng.randint(1, 8)), gating=rng.choice(("softmax", "sigmoid")), normalise=rng.random() < 0.7,
                scale=rng.choice((1.0, 1.0, 2.5)), bias=rng.random() < 0.4)
    if kind == "route":
        return {**case, "tokens": _log(rng, 1, 2000), "d": max(1, _log(rng, 512, 7000) // 32) * 32}
    up, down = rng.choice(("Q8_0", "Q4_0", "Q4_1", "Q4_K", "Q4_K", "Q5_K", "Q6_K")), rng.choice(("Q8_0", "Q4_0", "Q4_1", "Q4_K", "Q5_K", "Q6_K", "Q6_K"))
    both = up if BLOCK[up][1] == 256 else down  # (an FFN's length is a row of both kinds of weights)
    d = _length(rng, up if BLOCK[up][1] == 32 else "Q4_K", 512, 5120)
    ffn = min(_length(rng, both, 512, 14336), max(1, 8 * 14336 * 4096 // (experts * d) // 256) * 256)
    case = {**case, "d": d, "ffn": ffn, "up": up, "down": down, "tokens": rng.choice((1, rng.randint(2, 8), _log(rng, 9, 512))), "residual": rng.random() < 0.6,
            "activation": rng.choice(("silu", "silu", "gelu", "gelu_tanh", "relu"))}
    most = work(LARGEST)
    while case["tokens"] > 1 and (work(case)["bytes"] > most["bytes"] or work(case)["flops"] > most["flops"]):
        case["tokens"] = case["tokens"] * 3 // 4
    return case


# ------------------------------------------------------------------------------------------------- inputs


def _f16(v):
    return v.to(torch.float16).contiguous().view(torch.uint8).reshape(-1, 2)


def _nibbles(q):
    return (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8)


def _blocks(fmt, nb, gen):
    """nb blocks of the format as one uint8 tensor [nb, bytes], values about N(0, 0.02) as a quantiser of normal values makes them."""
    def u(count, lo, hi):
        return torch.empty(nb, count, device="cuda").uniform_(lo, hi, generator=gen)

    def ints(count, lo, hi):
        return torch.randint(lo, hi + 1, (nb, count), device="cuda", generator=gen)

    def quants(count, centre, spread, lo, hi):
        return torch.empty(nb, count, device="cuda").normal_(centre, spread, generator=gen).round_().clamp_(lo, hi).to(torch.int16)

    if fmt == "Q8_0":
        return torch.cat([_f16(u(1, 0.8, 1.2) * (0.02 / 56)), quants(32, 0.0, 56.0, -127, 127).to(torch.int8).view(torch.uint8)], 1)
    if fmt == "Q4_0":
        return torch.cat([_f16(u(1, 0.8, 1.2) * (0.02 / 3.5)), _nibbles(quants(32, 8.0, 3.5, 0, 15))], 1)
    if fmt == "Q4_1":
        d = u(1, 0.8, 1.2) * (0.02 / 3.5)
        return torch.cat([_f16(d), _f16(-7.5 * d), _nibbles(quants(32, 7.5, 3.5, 0, 15))], 1)
    if fmt in ("Q4_K", "Q5_K"):
        centre, spread = (7.5, 3.5) if fmt == "Q4_K" else (15.5, 7.0)
        d = u(1, 0.8, 1.2) * (0.02 / (spread * 52))
        sc, mn = ints(8, 42, 63), ints(8, 42, 63)  # eight 6-bit scales and minima in twelve bytes
        head = torch.cat([(sc[:, :4] | (sc[:, 4:] >> 4 << 6)), (mn[:, :4] | (mn[:, 4:] >> 4 << 6)), (sc[:, 4:] & 15) | ((mn[:, 4:] & 15) << 4)], 1).to(torch.uint8)
        q = quants(256, centre, spread, 0, 15 if fmt == "Q4_K" else 31)
        parts = [_f16(d), _f16(centre * d), head]
        if fmt == "Q5_K":
            bits = (q >> 4).reshape(nb, 8, 32)
            parts.append(sum(bits[:, i] << i for i in range(8)).to(torch.uint8))
        return torch.cat(parts + [_nibbles(q & 15)], 1)
    q = quants(256, 32.0, 16.0, 0, 63)  # Q6_K
    hi = (q >> 4).reshape(nb, 4, 64)
    qh = (hi[:, 0] | (hi[:, 1] << 2) | (hi[:, 2] << 4) | (hi[:, 3] << 6)).to(torch.uint8)
    sc = (ints(16, 70, 127) * (2 * ints(16, 0, 1) - 1)).to(torch.int8).view(torch.uint8)
    return torch.cat([_nibbles(q & 15), qh, sc, _f16(u(1, 0.8, 1.2) * (0.02 / (16 * 100)))], 1)


POOL_VALUES = 1 << 24  # (less fifteen blocks: a prime number of them, so that no two rows of a matrix begin alike)


def _weight(fmt, gen, *dims):
    """A weight [..., rows, blocks, bytes], cut from a pool of blocks."""
    _, qk, nb = BLOCK[fmt]
    need = math.prod(dims) // qk
    pool = _blocks(fmt, min(need, POOL_VALUES // qk - 15), gen)
    return pool.repeat(-(-need // pool.shape[0]), 1)[:need].contiguous().reshape(*dims[:-1], dims[-1] // qk, nb)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if own:
        import jitnn_amd
        jitnn_amd.init(0)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    s = dict(case=case)
    if case["kind"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        s["w"] = _weight(case["fmt"], gen, n, k)
        s["x"], s["y"] = randn(rows, k), torch.empty(rows, n, device="cuda")
        s["bias"] = 0.5 * randn(n) if case["bias"] else None
        s["residual"] = randn(rows, n) if case["residual"] else None
        if own:
            s["weight"] = jitnn_amd.Tensor.wrap_dev(jitnn_amd.DType[case["fmt"]], s["w"].data_ptr(), n, k)
        return s
    tokens, experts, d = case["tokens"], case["experts"], case["d"]
    s["x"] = randn(tokens, d)
    s["router"] = randn(experts, d) / math.sqrt(d)
    s["selection"] = 0.1 * randn(experts) if case["bias"] else None
    s["ids"] = torch.empty(tokens, case["used"], device="cuda", dtype=torch.int32)
    s["weights"] = torch.empty(tokens, case["used"], device="cuda")
    if case["kind"] == "moe":
        ffn = case["ffn"]
        s["gate"], s["up"], s["down"] = _weight(case["up"], gen, experts, ffn, d), _weight(case["up"], gen, experts, ffn, d), _weight(case["down"], gen, experts, d, ffn)
        s["y"] = torch.empty(tokens, d, device="cuda")
        s["residual"] = randn(tokens, d) if case["residual"] else None
    if own:
        router = jitnn_amd.Router(s["router"].cpu().numpy(), case["used"], gating=case["gating"], normalise=case["normalise"], scale=case["scale"],
                                  selection_bias=None if s["selection"] is None else s["selection"].cpu().numpy())
        s["plan"] = router
        if case["kind"] == "moe":
            up, down = jitnn_amd.DType[case["up"]], jitnn_amd.DType[case["down"]]
            s["plan"] = jitnn_amd.Moe(router, jitnn_amd.Tensor.wrap_dev(up, s["gate"].data_ptr(), experts, ffn, d),
                                      jitnn_amd.Tensor.wrap_dev(up, s["up"].data_ptr(), experts, ffn, d),
                                      jitnn_amd.Tensor.wrap_dev(down, s["down"].data_ptr(), experts, d, ffn), activation=case["activation"])
        s["workspace"] = torch.empty(max(16, s["plan"].workspace(tokens)), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------- the plain forms


def _half(b):
    """Pairs of bytes [..., 2 n] as n FP16 values, in FP32."""
    return b.contiguous().view(torch.float16).float()


def _scales(b):
    """The eight 6-bit scales and the eight minima of the bytes 4 .. 15 of a Q4_K / Q5_K block."""
    p, q, r = b[..., 4:8], b[..., 8:12], b[..., 12:16]
    return torch.cat([p & 63, (r & 15) | (p >> 6 << 4)], -1).float(), torch.cat([q & 63, (r >> 4) | (q >> 6 << 4)], -1).float()


def _values(fmt, w):
    """A weight [..., rows, blocks, bytes] as FP32 values [..., rows, k]."""
    def halves(b):  # bytes whose low nibbles come before their high ones
        return torch.cat([b & 15, b >> 4], -1).float()

    if fmt == "Q8_0":
        v = _half(w[..., :2]) * w[..., 2:].contiguous().view(torch.int8).float()
    elif fmt == "Q4_0":
        v = _half(w[..., :2]) * (halves(w[..., 2:]) - 8.0)
    elif fmt == "Q4_1":
        v = _half(w[..., :2]) * halves(w[..., 4:]) + _half(w[..., 2:4])
    elif fmt in ("Q4_K", "Q5_K"):
        sc, mn = _scales(w)
        qs = w[..., 16 if fmt == "Q4_K" else 48:].reshape(*w.shape[:-1], 4, 1, 32)
        q = torch.cat([qs & 15, qs >> 4], -2).reshape(*w.shape[:-1], 8, 32)
        if fmt == "Q5_K":
            shift = torch.arange(8, device=w.device, dtype=torch.uint8)[:, None]
            q = q | ((w[..., None, 16:48] >> shift & 1) << 4)
        v = q.float() * (_half(w[..., :2]) * sc)[..., None] - (_half(w[..., 2:4]) * mn)[..., None]
    else:  # Q6_K
        ql, qh = w[..., :128].reshape(*w.shape[:-1], 2, 2, 32), w[..., 128:192].reshape(*w.shape[:-1], 2, 1, 32)
        low = torch.cat([ql & 15, ql >> 4], -2)
        high = torch.cat([qh & 3, qh >> 2 & 3, qh >> 4 & 3, qh >> 6], -2)
        q = ((low | high << 4).float() - 32.0).reshape(*w.shape[:-1], 16, 16)
        v = q * (_half(w[..., 208:]) * w[..., 192:208].contiguous().view(torch.int8).float())[..., None]
    return v.reshape(*w.shape[:-2], -1)


def _act(kind, v):
    if kind == "relu":
        return v.clamp(min=0)
    if kind == "silu":
        return v / (1 + torch.exp(-v))
    if kind == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain_route(case, s):
    """In 64 bits: the sums are long, and an expert next to a border has to be chosen or left by both sides."""
    logits = s["x"].double() @ s["router"].double().t()
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True) if case["gating"] == "softmax" else 1 / (1 + torch.exp(-logits))
    by = logits if s["selection"] is None else p + s["selection"].double()
    ids = torch.sort(by, dim=1, descending=True, stable=True).indices[:, :case["used"]]  # (stable: ties go to the lowest index)
    w = torch.gather(p, 1, ids)
    if case["normalise"]:
        w = w / w.sum(1, keepdim=True)
    s["ids"].copy_(ids)
    s["weights"].copy_(w * case["scale"])
    return s["ids"], s["weights"]


def _plain_moe(case, s):
    ids, weights = _plain_route(case, s)
    tokens, experts, used, x = case["tokens"], case["experts"], case["used"], s["x"]
    if tokens * used <= experts:  # few tokens: their own experts' weights, a copy for each use
        at = ids.reshape(-1).long()
        xs = x.repeat_interleave(used, 0)[:, :, None]
        h = _act(case["activation"], torch.bmm(_values(case["up"], s["gate"][at]), xs)) * torch.bmm(_values(case["up"], s["up"][at]), xs)
        each = torch.bmm(_values(case["down"], s["down"][at]), h).reshape(tokens, used, -1)
        y = (each * weights[:, :, None]).sum(1)
    else:  # every expert on every token, most of them with weight 0
        share = torch.zeros(tokens, experts, device="cuda").scatter_add_(1, ids.long(), weights)
        xs = x.t().expand(experts, -1, -1).contiguous()
        h = _act(case["activation"], torch.bmm(_values(case["up"], s["gate"]), xs)) * torch.bmm(_values(case["up"], s["up"]), xs)
        y = torch.bmm(_values(case["down"], s["down"]), h * share.t()[:, None, :]).sum(0).t()
    s["y"].copy_(y if s["residual"] is None else y + s["residual"])
    return s["y"]


def _plain_linear(case, s):
    y = s["x"] @ _values(case["fmt"], s["w"]).t()
    y = _act(case["activation"], y if s["bias"] is None else y + s["bias"])
    s["y"].copy_(y if s["residual"] is None else y + s["residual"])
    return s["y"]


# ------------------------------------------------------------------------------------------------- the passes


def _at(t):
    return 0 if t is None else t.data_ptr()


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"route": _plain_route, "moe": _plain_moe, "linear": _plain_linear}[kind](case, s)
    if kind == "route":
        s["plan"].route_dev(s["x"].data_ptr(), case["tokens"], s["ids"].data_ptr(), s["weights"].data_ptr(), s["workspace"].data_ptr(), s["workspace"].numel())
        return s["ids"], s["weights"]
    if kind == "moe":
        s["plan"].layer_dev(s["x"].data_ptr(), case["tokens"], s["y"].data_ptr(), s["workspace"].data_ptr(), s["workspace"].numel(), residual_ptr=_at(s["residual"]))
        return s["y"]
    import jitnn_amd
    jitnn_amd.linear_dev(s["weight"], s["x"].data_ptr(), case["rows"], s["y"].data_ptr(), bias_ptr=_at(s["bias"]), activation=case["activation"],
                         residual_ptr=_at(s["residual"]))
    return s["y"]


# ------------------------------------------------------------------------------------------------- what a pass cannot do without


def _nbytes(fmt, values):
    _, qk, nb = BLOCK[fmt]
    return values // qk * nb


def work(case):
    if case["kind"] == "linear":
        n, k, rows = case["n"], case["k"], case["rows"]
        return dict(bytes=_nbytes(case["fmt"], n * k) + 4 * rows * k + 4 * rows * n * (2 if case["residual"] else 1) + (4 * n if case["bias"] else 0), flops=2 * rows * n * k)
    tokens, experts, used, d = case["tokens"], case["experts"], case["used"], case["d"]
    route = dict(bytes=4 * (experts * d + tokens * d) + 8 * tokens * used, flops=2 * tokens * experts * d)
    if case["kind"] == "route":
        return route
    # experts that so many tokens choose at all, where each is as likely as any other
    met = experts * (1 - (1 - used / experts) ** tokens)
    each = 2 * _nbytes(case["up"], case["ffn"] * d) + _nbytes(case["down"], case["ffn"] * d)
    return dict(bytes=int(4 * experts * d + met * each + 4 * tokens * d * (3 if case["residual"] else 2)), flops=route["flops"] + 6 * tokens * used * d * case["ffn"])


# ------------------------------------------------------------------------------------------------- in 64 bits, from the definitions


def _exact_values(fmt, w):
    """Values [rows, k] in 64 bits of blocks [rows, blocks, bytes], one place of a block after the other."""
    nb, qk = w.shape[1], BLOCK[fmt][1]
    out = torch.empty(w.shape[0], nb, qk, device="cuda", dtype=torch.float64)
    b = w.to(torch.int64)

    def half(i):
        bits = (b[..., i] | b[..., i + 1] << 8).to(torch.int32)
        return torch.where(bits >= 32768, bits - 65536, bits).to(torch.int16).view(torch.float16).double()

    def signed(v):
        return (v - (v >= 128) * 256).double()

    for e in range(qk):
        if fmt == "Q8_0":
            out[..., e] = half(0) * signed(b[..., 2 + e])
        elif fmt == "Q4_0":
            out[..., e] = half(0) * ((b[..., 2 + e % 16] >> 4 * (e // 16) & 15) - 8).double()
        elif fmt == "Q4_1":
            out[..., e] = half(0) * (b[..., 4 + e % 16] >> 4 * (e // 16) & 15).double() + half(2)
        elif fmt in ("Q4_K", "Q5_K"):
            j, l = e // 32, e % 32
            if j < 4:
                sc, mn = b[..., 4 + j] & 63, b[..., 8 + j] & 63
            else:
                sc = (b[..., 8 + j] & 15) + 16 * (b[..., j] >> 6)
                mn = (b[..., 8 + j] >> 4) + 16 * (b[..., 4 + j] >> 6)
            q = b[..., (16 if fmt == "Q4_K" else 48) + 32 * (j // 2) + l] >> 4 * (j % 2) & 15
            if fmt == "Q5_K":
                q = q + 16 * (b[..., 16 + l] >> j & 1)
            out[..., e] = half(0) * sc.double() * q.double() - half(2) * mn.double()
        else:
            n, j, l = e // 128, e // 32 % 4, e % 32
            q = (b[..., 64 * n + 32 * (j % 2) + l] >> 4 * (j // 2) & 15) + 16 * (b[..., 128 + 32 * n + l] >> 2 * j & 3)
            out[..., e] = half(208) * signed(b[..., 192 + e // 16]) * (q - 32).double()
    return out.reshape(w.shape[0], nb * qk)


def _exact_act(kind, v):
    return {None: lambda z: z, "relu": torch.relu, "silu": lambda z: z * torch.sigmoid(z), "gelu": lambda z: z * torch.special.ndtr(z),
            "gelu_tanh": lambda z: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))}[kind](v)


def _exact_route(case, s):
    z = (s["x"].double()[:, None, :] * s["router"].double()[None]).sum(2) if case["tokens"] * case["experts"] * case["d"] < 1 << 26 else \
        torch.nn.functional.linear(s["x"].double(), s["router"].double())
    p = torch.softmax(z, 1) if case["gating"] == "softmax" else torch.sigmoid(z)
    left = z.clone() if s["selection"] is None else p + s["selection"].double()
    ids, w = [], []
    for _ in range(case["used"]):
        best = left.amax(1, keepdim=True)
        i = (left == best).to(torch.uint8).argmax(1, keepdim=True)
        ids.append(i)
        w.append(torch.gather(p, 1, i))
        left.scatter_(1, i, -math.inf)
    ids, w = torch.cat(ids, 1), torch.cat(w, 1)
    return ids, case["scale"] * (w / w.sum(1, keepdim=True) if case["normalise"] else w)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["kind"] == "linear":
        y = _exact_act(case["activation"], x @ _exact_values(case["fmt"], s["w"]).t() + (0.0 if s["bias"] is None else s["bias"].double()))
        return y + (0.0 if s["residual"] is None else s["residual"].double())
    ids, w = _exact_route(case, s)
    if case["kind"] == "route":
        return None, w
    y = torch.zeros_like(x) if s["residual"] is None else s["residual"].double().clone()
    gate, up, down = (_exact_values(fmt, w.flatten(0, 1)).reshape(w.shape[0], w.shape[1], -1) for fmt, w in
                      ((case["up"], s["gate"]), (case["up"], s["up"]), (case["down"], s["down"])))
    for e in range(case["experts"]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel():
            h = _exact_act(case["activation"], x[t] @ gate[e].t()) * (x[t] @ up[e].t())
            y.index_add_(0, t, (h @ down[e].t()) * w[t, j][:, None])
    return y
