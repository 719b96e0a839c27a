"""The operators at the model's two token ends and its attention over an 8-bit cache, as measurable cases.

* ``logprob``   log probabilities of given tokens, their entropy and the top alternatives, from
                logits; in training with the gradient of the logits;
* ``embed``     the scaled embedding lookup; in training with the gradient of the table;
* ``decode`` ``extend`` ``prefill``  attention over a cache held in 8 bits, with one scale for each
                64 tokens and head: one token per sequence, more rows onto a filled cache, a prompt
                into an empty one. The cache takes the call's new rows.

With ``own`` false a pass computes the plain form: elementary torch operations in float32 (the
cache's rounding to 8 bits by the same formula, so its codes are equal bit for bit). With ``own``
true it makes the package's public calls. ``exact(case, seed)`` is the result in float64.
Import it with the repository's root as the working directory.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
BLOCK = 64                       # tokens that share a scale
HEADS = (8, 10, 12, 16)          # the model sizes' head counts; hidden = heads * 128
VOCABS = (32000, 50257, 65536, 131072)
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
CODE_MAX = {"e4m3": 448.0, "int8": 127.0}
IGNORE = -100


def listed():
    return [
        # one step of a small serving batch: the chosen tokens' log probabilities and five alternatives
        dict(name="logprob_step", kind="logprob", rows=4, V=65536, dtype="bf16", top=5, entropy=False, train=False,
             ignored=0.0),
        # scoring a document: every token's log probability, the entropy and eight alternatives; an
        # odd vocabulary, so rows start at any 2 bytes
        dict(name="logprob_score", kind="logprob", rows=1021, V=50257, dtype="bf16", top=8, entropy=True, train=False,
             ignored=0.0),
        # the loss of a training step over packed samples whose prompts do not count
        dict(name="logprob_train", kind="logprob", rows=8192, V=65536, dtype="bf16", top=0, entropy=False, train=True,
             ignored=0.25),
        # a policy step: float32 logits, log probabilities and entropy with their gradients
        dict(name="logprob_policy", kind="logprob", rows=2047, V=32000, dtype="f32", top=0, entropy=True, train=True,
             ignored=0.0),
        # the ids of one decode step
        dict(name="embed_step", kind="embed", T=64, V=65536, D=2048, table="bf16", out="bf16", train=False),
        # a training step: a float32 table, bfloat16 activations, and the table's gradient
        dict(name="embed_train", kind="embed", T=16384, V=65536, D=2048, table="f32", out="bf16", train=True),
        # the same for a small model in bfloat16, an odd number of tokens and an odd vocabulary
        dict(name="embed_train_small", kind="embed", T=4999, V=50257, D=1280, table="bf16", out="bf16", train=True),
        # one user: latency
        dict(name="decode_single", kind="decode", code="e4m3", B=1, S=1, H=16, Smax=1536, fill=0.6, len_seed=2, causal=False),
        # a full serving batch, each sequence at its own length
        dict(name="decode_batch", kind="decode", code="e4m3", B=64, S=1, H=16, Smax=4096, fill=0.75, len_seed=1, causal=False),
        # a few long documents
        dict(name="decode_long", kind="decode", code="int8", B=4, S=1, H=12, Smax=32768, fill=0.7, len_seed=4, causal=False),
        # the next turn of four conversations
        dict(name="extend_turn", kind="extend", code="e4m3", B=4, S=45, H=16, Smax=4096, fill=0.5, len_seed=3, causal=True),
        # two prompts into an empty cache
        dict(name="prefill", kind="prefill", code="e4m3", B=2, S=1021, H=16, Smax=2048, fill=0.0, len_seed=0, causal=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("logprob", "logprob", "logprob", "embed", "embed", "decode", "decode", "decode", "extend", "prefill"))
    heads = rng.choice(HEADS)
    if kind == "logprob":
        V, dtype, train = rng.choice(VOCABS + (rng.randint(1000, 100000),)), rng.choice(("bf16", "bf16", "f32")), rng.random() < 0.5
        most = min(8192, (8192 * 65536 if dtype == "bf16" else 2048 * 65536) // V)
        return dict(kind=kind, rows=_log_int(rng, 1, most), V=V, dtype=dtype, top=0 if train else rng.choice((0, 1, 5, 8, 20)),
                    entropy=rng.random() < 0.5, train=train, ignored=rng.choice((0.0, 0.3)))
    if kind == "embed":
        return dict(kind=kind, T=_log_int(rng, 1, 16384), V=rng.choice(VOCABS[:3] + (rng.randint(1000, 60000),)), D=128 * heads,
                    table=rng.choice(("bf16", "f32")), out="bf16", train=rng.random() < 0.75)
    code = rng.choice(("e4m3", "int8"))
    if kind == "decode":
        B = _log_int(rng, 1, 64)
        return dict(kind=kind, code=code, B=B, S=1, H=heads, Smax=BLOCK * _log_int(rng, 2, min(512, 4096 // B)),
                    fill=rng.choice((0.3, 0.75, 1.0)), len_seed=rng.randrange(1 << 20), causal=False)
    if kind == "extend":
        B = rng.randint(1, 8)
        return dict(kind=kind, code=code, B=B, S=_log_int(rng, 2, 256), H=heads, Smax=BLOCK * _log_int(rng, 8, 128),
                    fill=rng.choice((0.3, 0.6)), len_seed=rng.randrange(1 << 20), causal=rng.random() < 0.7)
    S = _log_int(rng, 16, 2048)
    return dict(kind=kind, code=code, B=rng.randint(1, max(1, min(8, 4096 // S))), S=S, H=heads,
                Smax=BLOCK * (-(-S // BLOCK) + rng.choice((1, 8, 16))), fill=0.0, len_seed=0, causal=rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7fffffff)


def _randn(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _tokens(g, n, V):
    """n token ids whose frequencies fall as one over their rank, as a language's do; the ranks are
    spread over the vocabulary."""
    rank = torch.exp(torch.rand(n, generator=g, device=DEV, dtype=torch.float64) * math.log(V)).long().clamp_(1, V)
    return (rank * 7919) % V


def _lens(case):
    """Rows already in each sequence's cache; the new rows still fit."""
    g = torch.Generator().manual_seed(case["len_seed"])
    most = case["Smax"] - case["S"]
    top = max(1, min(most, int(case["Smax"] * case["fill"] * 1.3)))
    low = max(0, min(top - 1, int(case["Smax"] * case["fill"] * 0.7)))
    lens = torch.randint(low, top + 1, (case["B"],), generator=g, dtype=torch.int32)
    # pieces of a long prompt, more than a block each, come after whole blocks
    return lens // BLOCK * BLOCK if case["S"] > BLOCK else lens


def _quantize(x, code):
    """Blocks x [..., n, 64, D] float32 -> (codes of the same shape, scales [..., n]): the scale is
    the block's largest magnitude over the type's, at least the smallest normal float32."""
    scale = (x.abs().amax((-2, -1)) / CODE_MAX[code]).clamp_min(2.0 ** -126)
    y = x / scale[..., None, None]
    return (y.round() if code == "int8" else y).to(TYPES[code]), scale


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = dict(case=case)
    if kind == "logprob":
        rows, V = case["rows"], case["V"]
        # a trained model's logits: a few tokens well above the rest
        x = torch.randn(rows, V, generator=g, device=DEV)
        x = x.mul_(2.0).add_(torch.randn(V, generator=g, device=DEV))
        t = torch.randint(0, V, (rows,), generator=g, device=DEV)
        best = x.argmax(-1)
        t = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.5, best, t)
        s["logits"] = x.to(TYPES[case["dtype"]])
        s["targets"] = torch.where(torch.rand(rows, generator=g, device=DEV) < case["ignored"], IGNORE, t)
        if case["train"]:
            s["g"] = torch.randn(rows, generator=g, device=DEV) / rows
            s["h"] = torch.randn(rows, generator=g, device=DEV) / rows
            s["logits"].requires_grad_()
        return s
    if kind == "embed":
        T, V, D = case["T"], case["V"], case["D"]
        s["ids"] = _tokens(g, T, V)
        s["table"] = _randn(g, V, D, scale=D ** -0.5, dtype=TYPES[case["table"]])
        s["scale"] = math.sqrt(D)
        if case["train"]:
            s["dy"] = _randn(g, T, D, scale=1e-2, dtype=TYPES[case["out"]])
            s["table"].requires_grad_()
        return s
    B, S, H, Smax = case["B"], case["S"], case["H"], case["Smax"]
    s["q"], s["k"], s["v"] = _randn(g, B, S, H, 128), _randn(g, B, S, H, 128, scale=2.0), _randn(g, B, S, H, 128)
    for name, size in (("k", 2.0), ("v", 1.0)):
        # each head at a size of its own
        rows = _randn(g, B, H, Smax // BLOCK, BLOCK, 128, scale=size)
        rows = rows * (0.5 + torch.rand(B, H, 1, 1, 1, generator=g, device=DEV)).to(torch.bfloat16)
        codes, s[name + "_scale"] = _quantize(rows.float(), case["code"])
        s[name + "_codes"] = codes.view(B, H, Smax, 128)
        s[name + "_recent"] = _randn(g, B, H, 2 * BLOCK, 128, scale=size)
        del rows, codes
    s["lens"] = 0 if kind == "prefill" else _lens(case).to(DEV)
    return s


# ---- one pass: the plain forms ---------------------------------------------------------------
def _plain_logprob(s):
    case, t = s["case"], s["targets"]
    x = s["logits"].detach().float()
    counted = t != IGNORE
    rows = torch.arange(x.shape[0], device=DEV)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    lse = m + torch.log(e.sum(-1, keepdim=True))
    at = torch.where(counted, t, 0)
    out = {"logprob": torch.where(counted, x[rows, at] - lse[:, 0], 0.0)}
    if case["entropy"]:
        p = torch.exp(x - lse)
        out["entropy"] = lse[:, 0] - (p * x).sum(-1)
    if case["top"]:
        # the value's bits in an order of whole numbers, then the lower index first
        bits = x.view(torch.int32).long()
        order = (torch.where(bits < 0, -2147483648 - bits, bits) << 32) + (x.shape[1] - 1 - torch.arange(x.shape[1], device=DEV))
        ids = x.shape[1] - 1 - (torch.topk(order, case["top"], dim=-1).values & 0xffffffff)
        out["top_logprobs"], out["top_ids"] = torch.gather(x, 1, ids) - lse, ids
    if case["train"]:
        g = torch.where(counted, s["g"], 0.0)[:, None]
        p = torch.exp(x - lse)
        d = -g * p
        d[rows, at] += g[:, 0]
        if case["entropy"]:
            d -= s["h"][:, None] * p * (x - lse + out["entropy"][:, None])
        out["grad"] = d.to(s["logits"].dtype)
    return out


def _plain_embed(s):
    case, table = s["case"], s["table"].detach()
    out = {"out": (table[s["ids"]].float() * s["scale"]).to(TYPES[case["out"]])}
    if case["train"]:
        d = torch.zeros(table.shape, dtype=torch.float32, device=DEV)
        d.index_add_(0, s["ids"], s["dy"].float() * s["scale"])
        out["grad"] = d.to(table.dtype)
    return out


def _rows_now(s, name, lens):
    """[B, H, Smax, 128] twice: keys or values as the attention sees them (8-bit blocks, then the rows
    of the incomplete block and the new rows in bfloat16), and the bfloat16 rows alone."""
    case = s["case"]
    B, H, Smax, S = case["B"], case["H"], case["Smax"], case["S"]
    pos = torch.arange(Smax, device=DEV)
    n = lens[:, None, None, None]
    p = pos[None, None, :, None]
    given = s[name].transpose(1, 2)
    fresh = torch.gather(given, 2, (p - n).clamp(0, S - 1).expand(B, H, Smax, 128))
    exact_rows = torch.where(p >= n, fresh, s[name + "_recent"][:, :, pos % (2 * BLOCK)])
    seen = s[name + "_codes"].float().view(B, H, -1, BLOCK, 128) * s[name + "_scale"][..., None, None]
    return torch.where(p >= n // BLOCK * BLOCK, exact_rows.float(), seen.view(B, H, Smax, 128)), exact_rows


def _plain_attend(s):
    case = s["case"]
    B, H, Smax, S = case["B"], case["H"], case["Smax"], case["S"]
    lens = s["lens"] if case["kind"] != "prefill" else torch.zeros(B, dtype=torch.int32, device=DEV)
    lens = lens.long()
    pos = torch.arange(Smax, device=DEV)
    k, k_rows = _rows_now(s, "k", lens)
    v, v_rows = _rows_now(s, "v", lens)
    end = lens + S
    q = s["q"].transpose(1, 2).float() * 128 ** -0.5
    w = torch.matmul(q, k.transpose(2, 3).contiguous())
    see = pos[None, None, :] < end[:, None, None]
    if case["causal"]:
        see = see & (pos[None, None, :] <= (lens[:, None] + torch.arange(S, device=DEV))[:, :, None])
    w = torch.where(see[:, None], w, -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    out = torch.matmul(w, v) / w.sum(-1, keepdim=True)
    # the cache takes the rows: blocks that are complete now in 8 bits, the others as they are
    block = torch.arange(Smax // BLOCK, device=DEV)[None]
    full = (block >= (lens // BLOCK)[:, None]) & (block < (end // BLOCK)[:, None])
    # and the last 64 rows before the incomplete block and those in it stay in bfloat16 as well,
    # position p in slot p % 128; here: the position that each slot is for
    first = (end // BLOCK * BLOCK - BLOCK)[:, None]
    here = first + (torch.arange(2 * BLOCK, device=DEV)[None] - first) % (2 * BLOCK)
    new = ((here >= lens[:, None]) & (here < end[:, None]))[:, None, :, None]
    for name, rows in (("k", k_rows), ("v", v_rows)):
        codes, scale = _quantize(rows.float().view(B, H, -1, BLOCK, 128), case["code"])
        s[name + "_scale"] = torch.where(full[:, None], scale, s[name + "_scale"])
        old = s[name + "_codes"].view(torch.uint8).view(B, H, -1, BLOCK, 128)
        codes = torch.where(full[:, None, :, None, None], codes.view(torch.uint8), old)
        s[name + "_codes"] = codes.view(B, H, Smax, 128).view(TYPES[case["code"]])
        at = here.clamp(0, Smax - 1)[:, None, :, None].expand(B, H, 2 * BLOCK, 128)
        s[name + "_recent"] = torch.where(new, torch.gather(rows, 2, at), s[name + "_recent"])
    return dict(out=out.transpose(1, 2).contiguous().to(torch.bfloat16))


def _cache_of(s, to):
    """The cache as it is held: the 8-bit numbers beside the scales that they are multiples of (so
    that a pass does no work that its user would not), and the rows of the incomplete blocks."""
    for name in ("k_codes", "v_codes", "k_scale", "v_scale", "k_recent", "v_recent"):
        to[name] = s[name]
    return to


# ---- one pass ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind == "logprob":
            return _plain_logprob(s)
        if kind == "embed":
            return _plain_embed(s)
        return _cache_of(s, _plain_attend(s))
    prefixlm = _package()
    if kind == "logprob":
        r = prefixlm.token_logprobs(s["logits"], s["targets"], entropy=case["entropy"], top_k=case["top"], ignore_index=IGNORE)
        out = {"logprob": r.logprob}
        if case["entropy"]:
            out["entropy"] = r.entropy
        if case["top"]:
            out["top_logprobs"], out["top_ids"] = r.top_logprobs, r.top_ids
        if case["train"]:
            heads, given = ((r.logprob, r.entropy), (s["g"], s["h"])) if case["entropy"] else ((r.logprob,), (s["g"],))
            out["grad"], = torch.autograd.grad(heads, (s["logits"],), given)
        return out
    if kind == "embed":
        y = prefixlm.embedding(s["ids"], s["table"], s["scale"], dtype=TYPES[case["out"]])
        if not case["train"]:
            return {"out": y}
        grad, = torch.autograd.grad(y, (s["table"],), s["dy"])
        return {"out": y, "grad": grad}
    cache = prefixlm.KVCacheQ8(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], s["k_recent"], s["v_recent"])
    y = prefixlm.flash_attn_with_kvcache_q8(s["q"], cache, k=s["k"], v=s["v"], cache_seqlens=s["lens"], causal=case["causal"])
    return _cache_of(s, dict(out=y))


def _package():
    """The framework, found as its users find it: its folder on the path."""
    at = os.path.join(os.getcwd(), "hrm-text_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import prefixlm
    return prefixlm


# ---- what a pass cannot do without ------------------------------------------------------
def _distinct(T, V):
    """How many different ids T tokens hold, on average."""
    r = torch.arange(1, V, dtype=torch.float64)
    return int(-torch.expm1(T * torch.log1p(-torch.log1p(1.0 / r) / math.log(V))).sum())


def work(case):
    kind = case["kind"]
    if kind == "logprob":
        size = 2 if case["dtype"] == "bf16" else 4
        n = case["rows"] * case["V"]
        small = case["rows"] * (12 + 12 * case["top"] + (4 if case["entropy"] else 0) + (8 if case["train"] else 0))
        # the statistics are of a whole row, so the gradient has to read the logits again, unless
        # the chip holds them meanwhile: counted once, as an input; the gradient is written
        return dict(bytes=n * size * (2 if case["train"] else 1) + small, flops=n * (8 if case["train"] else 4))
    if kind == "embed":
        T, V, D = case["T"], case["V"], case["D"]
        size = 2 if case["table"] == "bf16" else 4
        moved = 8 * T + _distinct(T, V) * D * size + 2 * T * D
        if case["train"]:
            moved += 2 * T * D + V * D * size
        return dict(bytes=moved, flops=T * D * (3 if case["train"] else 1))
    B, S, H = case["B"], case["S"], case["H"]
    lens = [0] * B if kind == "prefill" else _lens(case).tolist()
    old = sum(n // BLOCK * (BLOCK * 128 + 4) + n % BLOCK * 256 for n in lens)
    new = sum(((n + S) // BLOCK - n // BLOCK) * (BLOCK * 128 + 4) + min(S, (n + S) % BLOCK + BLOCK) * 256 for n in lens)
    pairs = sum(S * n + S * (S + 1) // 2 if case["causal"] else S * (n + S) for n in lens)
    # the cached rows in, q, k, v in and out, the rows that the cache takes
    return dict(bytes=H * (2 * old + 2 * new + 4 * 256 * B * S), flops=4 * 128 * H * pairs)


# ---- the same outputs in float64 ------------------------------------------------------------
def _exact_logprob(case, s):
    x, t = s["logits"].detach(), s["targets"].tolist()
    V, top = case["V"], case["top"]
    out = {k: [] for k in ("logprob", "entropy", "top_logprobs", "top_ids", "grad")}
    for i in range(0, x.shape[0], 256):
        part = x[i:i + 256].double()
        logp = torch.log_softmax(part, -1)
        p = logp.exp()
        ent = -(p * logp).sum(-1)
        hot = torch.zeros_like(p)
        for r, a in enumerate(t[i:i + 256]):
            if a != IGNORE:
                hot[r, a] = 1.0
        counted = hot.sum(-1)
        out["logprob"].append((hot * logp).sum(-1))
        out["entropy"].append(ent)
        if top:
            value, at = torch.sort(part, dim=-1, descending=True, stable=True)
            out["top_logprobs"].append(torch.gather(logp, 1, at[:, :top]))
            out["top_ids"].append(at[:, :top])
        if case["train"]:
            g = s["g"][i:i + 256].double()
            d = g[:, None] * (hot - p * counted[:, None])
            if case["entropy"]:
                d = d - s["h"][i:i + 256].double()[:, None] * p * (logp + ent[:, None])
            out["grad"].append(d.float() if V * x.shape[0] > 1 << 28 else d)   # 4 GB in 64 bits
    wanted = ["logprob"] + ["entropy"] * case["entropy"] + ["top_logprobs", "top_ids"] * (top > 0) + ["grad"] * case["train"]
    return {k: torch.cat(out[k]) for k in wanted}


def _exact_embed(case, s):
    table, ids = s["table"].detach(), s["ids"]
    out = {"out": table[ids].double() * s["scale"]}
    if case["train"]:
        grad = torch.zeros(case["V"], case["D"], dtype=torch.float64, device=DEV)
        order = torch.argsort(ids, stable=True)
        sums = torch.cat((torch.zeros(1, case["D"], dtype=torch.float64, device=DEV), s["dy"][order].double().cumsum(0)))
        value, count = torch.unique_consecutive(ids[order], return_counts=True)
        stop = count.cumsum(0)
        grad[value] = (sums[stop] - sums[stop - count]) * s["scale"]
        out["grad"] = grad
    return out


def _exact_attend(case, s):
    B, S, H = case["B"], case["S"], case["H"]
    lens = [0] * B if case["kind"] == "prefill" else _lens(case).tolist()
    out = torch.empty(B, S, H, 128, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        held = n - n % BLOCK
        for h in range(H):
            rows = []
            for name in ("k", "v"):
                unit = s[name + "_scale"][b, h, :held // BLOCK].double().repeat_interleave(BLOCK)
                rows.append(torch.cat((s[name + "_codes"][b, h, :held].to(torch.float32).double() * unit[:, None],
                                       s[name + "_recent"][b, h, torch.arange(held, n, device=DEV) % (2 * BLOCK)].double(),
                                       s[name][b, :, h].double())))
            score = s["q"][b, :, h].double() @ rows[0].t() / math.sqrt(128)
            if case["causal"]:
                score = score.masked_fill(torch.ones(S, n + S, dtype=torch.bool, device=DEV).triu(n + 1), -math.inf)
            out[b, :, h] = torch.softmax(score, -1) @ rows[1]
    # what the cache holds afterwards are rounded numbers: it has no value in more bits
    return {"out": out, **{k: None for k in ("k_codes", "v_codes", "k_scale", "v_scale", "k_recent", "v_recent")}}


def exact(case, seed):
    s = prepare(case, seed)
    return {"logprob": _exact_logprob, "embed": _exact_embed}.get(case["kind"], _exact_attend)(case, s)
