"""The work of serving a batch with jitnn_amd, operator by operator: rotary positions (both pairings, part of a head, scaled for
long contexts), appending keys and values to a paged cache with the rotation on the way, attention of a batch over that cache
whose leading pages every sequence shares, and the verification of drafted tokens from given random numbers.

`own` False: the operators' plain form in elementary torch operations.  `own` True: the calls of the package.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # one token's query and key heads (32 + 8 of 128), deep into a long context: the smallest call
        dict(name="rope_1_interleaved", kind="rope", tokens=1, heads=40, hd=128, rot=128, interleaved=True, scaling="none", far=131072),
        # a prompt that fills a window of 4096, scaled for a context beyond the trained one
        dict(name="rope_4096_half_yarn", kind="rope", tokens=4096, heads=32, hd=128, rot=128, interleaved=False, scaling="yarn", far=32768),
        # one sequence, one token, FP32 cache, the heads of a small model
        dict(name="append_1_f32", kind="append", seqs=1, each=1, ragged=False, context=700, heads=8, kv=2, hd=64, rot=64, interleaved=True, scaling="none",
             page=16, type="f32"),
        # a batch of 64 decoding together, 32 query heads over 8 key / value heads of 128
        dict(name="append_64_f16", kind="append", seqs=64, each=1, ragged=False, context=2000, heads=32, kv=8, hd=128, rot=128, interleaved=False,
             scaling="yarn", page=64, type="f16"),
        # a prompt of 4096 tokens on its way into the cache
        dict(name="append_prompt_4096_f16", kind="append", seqs=1, each=4096, ragged=False, context=4096, heads=32, kv=8, hd=128, rot=128,
             interleaved=True, scaling="linear", page=64, type="f16"),
        # one sequence of a small model, nothing shared: the smallest attention
        dict(name="attention_1x600_f32", kind="attention", seqs=1, each=1, ragged=False, shared=0, suffix=600, heads=8, kv=2, hd=64, page=16, type="f32"),
        # eight sequences of a model without grouped heads, nothing shared, lengths of every size up to 2000
        dict(name="attention_8x2000_f16", kind="attention", seqs=8, each=1, ragged=False, shared=0, suffix=2000, heads=32, kv=32, hd=128, page=32, type="f16"),
        # 24 continuations of a prompt of about 1000, up to five tokens of each in a pass (drafts), in FP32
        dict(name="attention_24x5_drafts_f32", kind="attention", seqs=24, each=5, ragged=True, shared=62, suffix=401, heads=32, kv=8, hd=128, page=16,
             type="f32"),
        # 64 continuations of a long document: the largest
        dict(name="attention_64x16384_f16", kind="attention", seqs=64, each=1, ragged=False, shared=256, suffix=512, heads=32, kv=8, hd=128, page=64,
             type="f16"),
        # one sequence with four tokens drafted by lookup, a vocabulary of 32000
        dict(name="verify_1x5_lookup", kind="verify", seqs=1, each=5, ragged=False, vocab=32000, drafts="lookup"),
        # 16 sequences with up to eight looked-up tokens each, a vocabulary of 128256
        dict(name="verify_16x9_lookup", kind="verify", seqs=16, each=9, ragged=True, vocab=128256, drafts="lookup"),
        # 32 sequences with four tokens drawn from a draft model's probabilities
        dict(name="verify_32x5_model", kind="verify", seqs=32, each=5, ragged=False, vocab=128256, drafts="model"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


LARGEST = dict(kind="attention", seqs=64, each=1, ragged=False, shared=256, suffix=512, heads=32, kv=8, hd=128, page=64, type="f16")


def draw(rng):
    kind = rng.choices(("rope", "append", "attention", "verify"), (2, 3, 6, 3))[0]
    if kind == "verify":
        each, vocab = rng.randint(1, 9), _log(rng, 1000, 150000)
        seqs = min(_log(rng, 1, 64), max(1, 32 * 5 * 128256 // (each * vocab)))
        return dict(kind=kind, seqs=seqs, each=each, ragged=rng.random() < 0.5, vocab=vocab, drafts=rng.choice(("lookup", "model")))
    interleaved, scaling = rng.random() < 0.5, rng.choice(("none", "linear", "factors", "yarn"))
    if kind == "rope":
        hd = rng.choice((64, 80, 96, 128, 192, 256))
        rot = rng.choice((hd, hd, hd // 2, 32))
        heads = rng.randint(1, 64)
        tokens = min(_log(rng, 1, 8192), 4096 * 32 * 128 // (heads * hd))
        return dict(kind=kind, tokens=tokens, heads=heads, hd=hd, rot=rot, interleaved=interleaved, scaling=scaling, far=_log(rng, tokens + 1, 1000000))
    hd, kv, group = rng.choice((64, 128, 128, 192, 256)), rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 5, 7, 8))
    page, dtype = rng.choice((16, 32, 64, 128)), rng.choice(("f16", "f32"))
    if kind == "append":
        seqs = _log(rng, 1, 128)
        each = min(_log(rng, 1, 4096), max(1, 4096 * 38 * 128 // (seqs * kv * (group + 2) * hd)))
        return dict(kind=kind, seqs=seqs, each=each, ragged=rng.random() < 0.5, context=each + _log(rng, 1, 3000), heads=kv * group, kv=kv, hd=hd,
                    rot=rng.choice((hd, hd, hd // 2)), interleaved=interleaved, scaling=scaling, page=page, type=dtype)
    each = rng.choice((1, 1, 1, rng.randint(2, 8), rng.randint(2, 8), _log(rng, 16, 512)))
    seqs = _log(rng, 1, 64) if each <= 8 else rng.randint(1, 4)
    shared = rng.choice((0, _log(rng, 64, 16384), _log(rng, 64, 16384))) // page
    case = dict(kind=kind, seqs=seqs, each=each, ragged=rng.random() < 0.5, shared=shared, suffix=each + _log(rng, 1, 2000), heads=kv * group, kv=kv, hd=hd,
                page=page, type=dtype)
    most = work(LARGEST)
    while case["seqs"] > 1 and (work(case)["bytes"] > most["bytes"] or work(case)["flops"] > most["flops"]):
        case["seqs"] -= 1
    while case["shared"] > 0 and (work(case)["bytes"] > most["bytes"] or work(case)["flops"] > most["flops"]):
        case["shared"] //= 2
    return case


# ------------------------------------------------------------------------------------------------- inputs

BETA_FAST, BETA_SLOW, TRAINED, FACTOR, THETA = 32.0, 1.0, 8192, 4.0, 500000.0


def _counts(case):
    """Tokens of each sequence in this pass."""
    return [1 + (7 * i + case["each"] - 1) % case["each"] if case["ragged"] else case["each"] for i in range(case["seqs"])]


def _own_positions(case):
    """Positions of each sequence behind the shared ones, this pass's tokens among them: every length up to the longest."""
    return [max(n, -(-case["suffix"] * (i + 1) // case["seqs"])) for i, n in enumerate(_counts(case))]


def _frequencies(case):
    """The rotation's frequencies and magnitude, as a program computes them once for a model."""
    r = case["rot"]
    f = torch.pow(torch.tensor(THETA, dtype=torch.float64), -torch.arange(0, r, 2, dtype=torch.float64) / r)
    factors = 1.0 + 7.0 * torch.arange(r // 2, dtype=torch.float64) / (r // 2)
    if case["scaling"] == "linear":
        return f / FACTOR, 1.0, None
    if case["scaling"] == "factors":
        factors = factors.float()
        return f / factors.double(), 1.0, factors
    if case["scaling"] == "yarn":
        at = [r * math.log(TRAINED / (2 * math.pi * b)) / (2 * math.log(THETA)) for b in (BETA_FAST, BETA_SLOW)]
        lo, hi = max(0, math.floor(at[0])), min(r - 1, math.ceil(at[1]))
        ramp = ((torch.arange(r // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / FACTOR * ramp, 0.1 * math.log(FACTOR) + 1.0, None
    return f, 1.0, None


def _prepare_rope(case, s):
    f, s["magnitude"], factors = _frequencies(case)
    s["f"] = f.cuda()
    if own:
        import jitnn_amd
        kind = case["scaling"] if case["scaling"] in ("linear", "yarn") else None
        s["rope"] = jitnn_amd.Rope(case["rot"], theta=THETA, interleaved=case["interleaved"], scaling=kind, factor=FACTOR, original_context=TRAINED,
                                   beta_fast=BETA_FAST, beta_slow=BETA_SLOW, freq_factors=None if factors is None else factors.numpy())


def _prepare_cache(case, s, gen, positions, shared, room):
    """A pool of pages in the caller's memory, each sequence's pages anywhere in it, the leading `shared` ones everybody's, and
    `room` for so many positions behind them."""
    seqs, page, kv, hd = case["seqs"], case["page"], case["kv"], case["hd"]
    width = shared + -(-room // page)
    pages = shared + seqs * (width - shared) + 3
    kind = torch.float16 if case["type"] == "f16" else torch.float32
    s["k"] = torch.randn(pages, kv, page, hd, device="cuda", generator=gen).to(kind)
    s["v"] = torch.randn(pages, kv, page, hd, device="cuda", generator=gen).to(kind)
    ids = torch.randperm(pages, device="cuda", generator=gen)[: pages - 3].to(torch.int32)
    s["tables"] = torch.cat([ids[:shared].expand(seqs, shared), ids[shared:].reshape(seqs, width - shared)], 1).contiguous()
    counts = _counts(case)
    s["starts"] = torch.tensor([0] + np.cumsum(counts).tolist(), device="cuda", dtype=torch.int32)
    s["lens"] = torch.tensor([shared * page + p for p in positions], device="cuda", dtype=torch.int32)
    s["tokens"], s["each"], s["width"] = sum(counts), max(counts), width
    if own:
        import jitnn_amd
        s["cache"] = jitnn_amd.PagedCache.wrap_dev(s["k"].data_ptr(), s["v"].data_ptr(), 1, kv, hd, pages, page, 1 if case["type"] == "f16" else 0)
        s["batch"] = jitnn_amd.Batch(seqs, s["tokens"], s["each"], shared * page + max(positions), s["tables"].data_ptr(), width, s["starts"].data_ptr(),
                                     s["lens"].data_ptr(), shared)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if own:
        import jitnn_amd
        jitnn_amd.init(0)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    s = dict(case=case)
    kind = case["kind"]
    if kind == "rope":
        _prepare_rope(case, s)
        first = int(torch.randint(0, case["far"] - case["tokens"] + 1, (1,), device="cuda", generator=gen).item())
        s["positions"] = torch.arange(first, first + case["tokens"], device="cuda", dtype=torch.int32)
        s["x"] = randn(case["tokens"], case["heads"], case["hd"])
        s["y"] = torch.empty_like(s["x"])
    elif kind == "append":
        _prepare_rope(case, s)
        counts = _counts(case)
        behind = torch.randint(0, case["context"] - case["each"] + 1, (case["seqs"],), device="cuda", generator=gen).tolist()
        _prepare_cache(case, s, gen, [b + n for b, n in zip(behind, counts)], 0, case["context"])
        # (one buffer of the three projections, as a linear of all of them leaves it)
        s["qkv"] = randn(s["tokens"], (case["heads"] + 2 * case["kv"]) * case["hd"])
        s["q_out"] = torch.empty(s["tokens"], case["heads"], case["hd"], device="cuda")
    elif kind == "attention":
        _prepare_cache(case, s, gen, _own_positions(case), case["shared"], case["suffix"])
        s["q"] = randn(s["tokens"], case["heads"], case["hd"])
        s["y"] = torch.empty_like(s["q"])
        if own:
            s["workspace"] = torch.empty(max(16, s["cache"].attention_workspace(s["batch"], case["heads"])), dtype=torch.uint8, device="cuda")
    else:
        counts = _counts(case)
        rows, vocab = sum(counts), case["vocab"]
        s["starts"] = torch.tensor([0] + np.cumsum(counts).tolist(), device="cuda", dtype=torch.int32)
        s["each"] = max(counts)
        s["logits"] = 3 * randn(rows, vocab)
        # every fourth sequence is decoded greedily
        s["temperatures"] = torch.tensor([0.0 if i % 4 == 3 else 0.6 + 0.1 * (i % 5) for i in range(case["seqs"])], device="cuda")
        seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), torch.tensor(counts, device="cuda"))
        t = s["temperatures"][seq].where(s["temperatures"][seq] > 0, torch.ones_like(s["temperatures"][seq]))[:, None]
        q = torch.softmax((s["logits"] + 0.5 * randn(rows, vocab)) / t, 1)
        drawn = torch.multinomial(q, 1, generator=gen)[:, 0].to(torch.int32)
        s["tokens"] = torch.cat([torch.randint(0, vocab, (1,), device="cuda", generator=gen, dtype=torch.int32), drawn[:-1]])
        s["q"] = q if case["drafts"] == "model" else None
        s["uniforms"] = torch.rand(rows, 2, device="cuda", generator=gen)
        s["out"] = torch.empty(rows, device="cuda", dtype=torch.int32)
        s["accepted"] = torch.empty(case["seqs"], device="cuda", dtype=torch.int32)
        if own:
            import jitnn_amd
            s["workspace"] = torch.empty(max(16, jitnn_amd.verify_workspace(rows, case["seqs"], vocab)), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------- the plain forms


def _places(s):
    """Every token's sequence and position."""
    at = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].contiguous(), at.to(torch.int32), right=True)
    return seq, (s["lens"] - s["starts"][1:])[seq] + at


def _rotated(case, s, x, positions):
    """x [tokens, heads, hd] rotated: angles of far positions in 64 bits, the products in 32."""
    angle = positions.double()[:, None] * s["f"]
    cos, sin = ((g(angle) * s["magnitude"]).float()[:, None, :] for g in (torch.cos, torch.sin))
    r = case["rot"]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., : r // 2], x[..., r // 2:r])
    y = x.clone()
    if case["interleaved"]:
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, a * sin + b * cos
    else:
        y[..., : r // 2], y[..., r // 2:r] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_append(case, s):
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    q, k, v = s["qkv"].reshape(s["tokens"], heads + 2 * kv, hd).split((heads, kv, kv), 1)
    seq, pos = _places(s)
    page = s["tables"][seq, pos // case["page"]].long()
    at = pos % case["page"]
    s["q_out"].copy_(_rotated(case, s, q, pos))
    s["k"][page, :, at] = _rotated(case, s, k, pos).to(s["k"].dtype)
    s["v"][page, :, at] = v.to(s["v"].dtype)
    return s["q_out"], s["k"], s["v"]


def _plain_attention(case, s):
    """The shared positions' products for all rows at once, the others' sequence by sequence (padded to the longest)."""
    kv, hd, seqs, each = case["kv"], case["hd"], case["seqs"], s["each"]
    group, n = case["heads"] // kv, case["shared"] * case["page"]
    seq, pos = _places(s)
    at = (s["starts"][:-1, None] + torch.arange(each, device="cuda")).clamp(max=s["tokens"] - 1)  # [seqs, each]: padded ones repeat another
    q = (s["q"] * (1.0 / math.sqrt(hd))).reshape(s["tokens"], kv, group, hd)[at].permute(0, 2, 1, 3, 4).reshape(seqs, kv, each * group, hd)
    own_pages = s["tables"][:, case["shared"]:].long()
    k = s["k"][own_pages].transpose(1, 2).reshape(seqs, kv, -1, hd).float()
    v = s["v"][own_pages].transpose(1, 2).reshape(seqs, kv, -1, hd).float()
    scores = torch.matmul(q, k.transpose(2, 3).contiguous())
    if n:
        first = s["tables"][0, :case["shared"]].long()
        kp = s["k"][first].transpose(0, 1).reshape(kv, n, hd).float()
        vp = s["v"][first].transpose(0, 1).reshape(kv, n, hd).float()
        ahead = torch.matmul(q.transpose(0, 1).reshape(kv, seqs * each * group, hd), kp.transpose(1, 2).contiguous())
        scores = torch.cat([ahead.reshape(kv, seqs, each * group, n).transpose(0, 1), scores], 3)
    hidden = torch.arange(scores.shape[3], device="cuda") > pos[at].repeat_interleave(group, 1)[:, None, :, None]
    scores = scores.masked_fill(hidden, -math.inf)
    p = torch.exp(scores - scores.amax(3, keepdim=True))
    p = p / p.sum(3, keepdim=True)
    y = torch.matmul(p[..., n:], v)
    if n:
        y = y + torch.matmul(p[..., :n].transpose(0, 1).reshape(kv, seqs * each * group, n), vp).reshape(kv, seqs, each * group, hd).transpose(0, 1)
    y = y.reshape(seqs, kv, each, group, hd).transpose(1, 2).reshape(seqs, each, case["heads"], hd)
    at_all = torch.arange(s["tokens"], device="cuda") - s["starts"][:-1][seq]
    s["y"].copy_(y[seq, at_all])
    return s["y"]


def _plain_verify(case, s):
    """In 64 bits: the sums are long, and a draw next to a border has to fall on the same side."""
    seqs, each, starts = case["seqs"], s["each"], s["starts"].long()
    logits = s["logits"].double()
    rows = logits.shape[0]
    seq = torch.searchsorted(starts[1:].contiguous(), torch.arange(rows, device="cuda"), right=True)
    t = s["temperatures"].double()[seq][:, None]
    m, best = logits.max(1, keepdim=True)
    best = (logits == m).to(torch.uint8).argmax(1, keepdim=True)  # the lowest index among equal ones
    p = torch.exp((logits - m) / t.where(t > 0, torch.ones_like(t)))
    p = (p / p.sum(1, keepdim=True)).where(t > 0, torch.zeros_like(p).scatter_(1, best, 1.0))
    count = starts[1:] - starts[:-1]
    j = torch.arange(each, device="cuda")
    at = (starts[:-1, None] + j).clamp(max=rows - 1)
    x = s["tokens"].long()[(at + 1).clamp(max=rows - 1)]
    drafted = j < count[:, None] - 1
    qx = s["q"][at, x].double() if s["q"] is not None else torch.ones_like(s["uniforms"][:, 0].double()[at])
    kept = drafted & (s["uniforms"][:, 0].double()[at] * qx < p[at, x])
    accepted = kept.long().cumprod(1).sum(1)
    r = starts[:-1] + accepted
    refused = (accepted < count - 1)[:, None]
    if s["q"] is not None:
        rest = (p[r] - s["q"][r].double()).clamp(min=0)
    else:
        rest = p[r].scatter(1, s["tokens"].long()[(r + 1).clamp(max=rows - 1)][:, None], 0.0)
    sums = rest.where(refused, p[r]).cumsum(1)
    drawn = (sums <= s["uniforms"][:, 1].double()[r][:, None] * sums[:, -1:]).sum(1).clamp(max=case["vocab"] - 1)
    s["out"].fill_(-1)
    local = torch.arange(rows, device="cuda") - starts[:-1][seq]
    following = s["tokens"][(torch.arange(rows, device="cuda") + 1).clamp(max=rows - 1)]
    s["out"].copy_(following.where(local < accepted[seq], s["out"]))
    s["out"][r] = drawn.to(torch.int32)
    s["accepted"].copy_(accepted)
    return s["out"], s["accepted"]


# ------------------------------------------------------------------------------------------------- the passes


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind == "rope":
            s["y"].copy_(_rotated(case, s, s["x"], s["positions"]))
            return s["y"]
        return {"append": _plain_append, "attention": _plain_attention, "verify": _plain_verify}[kind](case, s)
    if kind == "rope":
        s["rope"].apply_dev(s["x"].data_ptr(), s["positions"].data_ptr(), case["tokens"], case["heads"], case["hd"], s["y"].data_ptr())
        return s["y"]
    if kind == "append":
        heads, kv, hd = case["heads"], case["kv"], case["hd"]
        q, row = s["qkv"].data_ptr(), (heads + 2 * kv) * hd
        s["cache"].append_dev(0, s["batch"], s["rope"], heads, q, s["q_out"].data_ptr(), q + 4 * heads * hd, q + 4 * (heads + kv) * hd, q_stride=row,
                              q_out_stride=heads * hd, k_stride=row, v_stride=row)
        return s["q_out"], s["k"], s["v"]
    if kind == "attention":
        s["cache"].attention_dev(0, s["batch"], case["heads"], s["q"].data_ptr(), 1.0 / math.sqrt(case["hd"]), s["y"].data_ptr(), s["workspace"].data_ptr(),
                                 s["workspace"].numel())
        return s["y"]
    import jitnn_amd
    q = s["q"]
    jitnn_amd.verify_drafts_dev(s["logits"].data_ptr(), s["logits"].shape[0], case["vocab"], s["starts"].data_ptr(), case["seqs"], s["tokens"].data_ptr(),
                                s["temperatures"].data_ptr(), s["uniforms"].data_ptr(), s["out"].data_ptr(), s["accepted"].data_ptr(),
                                s["workspace"].data_ptr(), s["workspace"].numel(), draft_probs_ptr=0 if q is None else q.data_ptr())
    return s["out"], s["accepted"]


# ------------------------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    kind = case["kind"]
    if kind == "rope":
        values = case["tokens"] * case["heads"] * case["hd"]
        return dict(bytes=8 * values + 4 * case["tokens"], flops=3 * values)
    if kind == "verify":
        rows = sum(_counts(case))
        return dict(bytes=4 * rows * case["vocab"] + (4 * case["seqs"] * case["vocab"] if case["drafts"] == "model" else 0), flops=4 * rows * case["vocab"])
    size = 2 if case["type"] == "f16" else 4
    tokens, row = sum(_counts(case)), case["kv"] * case["hd"]
    if kind == "append":
        q = case["heads"] * case["hd"]
        return dict(bytes=tokens * (8 * q + 8 * row + 2 * size * row), flops=3 * tokens * (q + row))
    n, positions = case["shared"] * case["page"], _own_positions(case)
    pairs = sum(c * (n + p) - c * (c - 1) // 2 for c, p in zip(_counts(case), positions))
    return dict(bytes=2 * size * row * (n + sum(positions)) + 8 * tokens * case["heads"] * case["hd"], flops=4 * case["heads"] * case["hd"] * pairs)


# ------------------------------------------------------------------------------------------------- in 64 bits, from the definitions


def _exact_angles(case, positions):
    """cos and sin [tokens, rot / 2], with the magnitude, of whole positions."""
    r = case["rot"]
    f = np.array([THETA ** (-2.0 * i / r) for i in range(r // 2)])
    magnitude = 1.0
    if case["scaling"] == "linear":
        f = f / FACTOR
    elif case["scaling"] == "factors":
        f = f / np.array([np.float32(1.0 + 7.0 * i / (r // 2)) for i in range(r // 2)], dtype=np.float64)
    elif case["scaling"] == "yarn":
        lo = max(0, math.floor(r * math.log(TRAINED / (2 * math.pi * BETA_FAST)) / (2 * math.log(THETA))))
        hi = min(r - 1, math.ceil(r * math.log(TRAINED / (2 * math.pi * BETA_SLOW)) / (2 * math.log(THETA))))
        for i in range(r // 2):
            g = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f[i] = (1 - g) * f[i] + g * f[i] / FACTOR
        magnitude = 1.0 + 0.1 * math.log(FACTOR)
    angle = np.outer(np.asarray(positions, dtype=np.float64), f)
    return torch.from_numpy(magnitude * np.cos(angle)).cuda(), torch.from_numpy(magnitude * np.sin(angle)).cuda()


def _exact_rotation(case, x, positions):
    c, d = _exact_angles(case, positions)
    x = x.double()
    y = x.clone()
    r = case["rot"]
    for i in range(r // 2):
        i0, i1 = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
        y[:, :, i0] = x[:, :, i0] * c[:, i, None] - x[:, :, i1] * d[:, i, None]
        y[:, :, i1] = x[:, :, i0] * d[:, i, None] + x[:, :, i1] * c[:, i, None]
    return y


def _positions_of(s):
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    return [(i, lens[i] - (starts[i + 1] - starts[i]) + j) for i in range(len(lens)) for j in range(starts[i + 1] - starts[i])]


def _exact_append(case, s):
    heads, kv, hd, page = case["heads"], case["kv"], case["hd"], case["page"]
    x = s["qkv"].reshape(s["tokens"], heads + 2 * kv, hd)
    places = _positions_of(s)
    rotated = _exact_rotation(case, x[:, :heads + kv], [p for _, p in places])
    k, v, tables = s["k"].double(), s["v"].double(), s["tables"].cpu()
    ids = torch.tensor([int(tables[i, p // page]) for i, p in places], device="cuda")
    at = torch.tensor([p % page for _, p in places], device="cuda")
    k[ids, :, at] = rotated[:, heads:]
    v[ids, :, at] = x[:, heads + kv:].double()
    return rotated[:, :heads].contiguous(), k, v


def _exact_attention(case, s):
    kv, hd, page = case["kv"], case["hd"], case["page"]
    group = case["heads"] // kv
    y = torch.zeros(s["tokens"], case["heads"], hd, device="cuda", dtype=torch.float64)
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    for i in range(case["seqs"]):
        ids = s["tables"][i, : -(-lens[i] // page)].long()
        k = s["k"][ids].permute(1, 0, 2, 3).reshape(kv, -1, hd)[:, : lens[i]].double()
        v = s["v"][ids].permute(1, 0, 2, 3).reshape(kv, -1, hd)[:, : lens[i]].double()
        a, b = starts[i], starts[i + 1]
        q = s["q"][a:b].double().reshape(b - a, kv, group, hd).permute(1, 2, 0, 3).reshape(kv, group * (b - a), hd)
        z = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(hd)
        limit = torch.arange(lens[i] - (b - a), lens[i], device="cuda").repeat(group)
        z[:, torch.arange(lens[i], device="cuda")[None, :] > limit[:, None]] = -math.inf
        o = torch.bmm(torch.softmax(z, 2), v)
        y[a:b] = o.reshape(kv, group, b - a, hd).permute(2, 0, 1, 3).reshape(b - a, case["heads"], hd)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rotation(case, s["x"], s["positions"].tolist())
    if case["kind"] == "append":
        return _exact_append(case, s)
    if case["kind"] == "attention":
        return _exact_attention(case, s)
    return None  # (whole numbers only)
