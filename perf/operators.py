"""The measured operators of the paged key/value cache: what writes it (`ops.paged_append`) and what reads it (`ops.paged_attention`).

A case is a dict of plain values:
  op        "append" or "attend"
  batch     sequences of the call; `rows` the most new rows of one (1: a decoding step), `rows_lo` the fewest
  held_lo, held   tokens that the cache holds of a sequence before the call: the fewest and the most
  heads, kv_heads, head_dim, page (tokens), kind "e4m3" (8 bits, one scale per page and head) or "bf16"
  qk_norm   append: a norm of each q and k head before the rotation
  window, causal  attend: the sliding window (0: none), and whether a row sees the keys behind it
The sequences' lengths lie evenly (over the logarithm) between the fewest and the most; the seed says which sequence has which.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
LEAST_EXPONENT = -60
EPS = 1e-5


def _case(name, op, batch, rows_lo, rows, held_lo, held, heads, kv_heads, head_dim, page, kind, qk_norm=False, window=0, causal=True):
    c = {"name": name, "op": op, "batch": batch, "rows_lo": rows_lo, "rows": rows, "held_lo": held_lo, "held": held, "heads": heads,
         "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "kind": kind}
    return c | ({"qk_norm": qk_norm} if op == "append" else {"window": window, "causal": causal})


def listed():
    return [
        # one user's next token, 7B-class heads
        _case("append_chat", "append", 1, 1, 1, 437, 437, 32, 8, 128, 64, "e4m3"),
        # a decoding step of a full serving batch, sequences of all lengths
        _case("append_step", "append", 64, 1, 1, 1, 4000, 32, 8, 128, 64, "e4m3"),
        # prompts of several users going in at once, some behind a shared history
        _case("append_prompts", "append", 7, 130, 2048, 0, 777, 32, 8, 128, 64, "e4m3"),
        # the retriever's heads with QK-norm, unquantised pages of another size
        _case("append_norm", "append", 24, 33, 301, 0, 50, 8, 4, 64, 32, "bf16", qk_norm=True),
        # one user chatting
        _case("decode_chat", "attend", 1, 1, 1, 501, 501, 32, 8, 128, 64, "e4m3"),
        # a full serving batch
        _case("decode_batch", "attend", 64, 1, 1, 37, 8191, 32, 8, 128, 64, "e4m3"),
        # as many kv heads as query heads, head_dim 64, unquantised
        _case("decode_heads", "attend", 32, 1, 1, 300, 2047, 16, 16, 64, 16, "bf16"),
        # one long document
        _case("decode_long", "attend", 1, 1, 1, 100003, 100003, 32, 8, 128, 128, "e4m3"),
        # the sliding window of the 7B preset behind longer sequences
        _case("decode_window", "attend", 12, 1, 1, 2500, 16000, 32, 8, 128, 64, "bf16", window=4096),
        # drafted tokens of a few users being verified
        _case("drafts", "attend", 8, 2, 4, 900, 4000, 32, 8, 128, 64, "e4m3"),
        # a chunk of a long prompt behind what the cache holds of it
        _case("chunk", "attend", 1, 512, 512, 7500, 7500, 32, 8, 128, 64, "e4m3"),
        # prompts of several users at once
        _case("prompts", "attend", 6, 200, 2048, 0, 700, 32, 8, 128, 64, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    largest = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= largest["bytes"] and w["flops"] <= largest["flops"]:
            return c


def _draw(rng):
    op = rng.choice(["append", "append", "decode", "decode", "decode", "drafts", "chunk"])
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (32, 32, 128), (16, 16, 64), (8, 4, 64), (12, 12, 128), (16, 1, 128), (8, 2, 64)])
    kind, page = rng.choice(["e4m3", "e4m3", "bf16"]), rng.choice([16, 32, 64, 64, 128])
    batch = _log_int(rng, 1, 64)
    if op == "append":
        rows = rng.choice([1, _log_int(rng, 2, max(2, min(2048, 8192 // batch)))])
        held = _log_int(rng, 1, 4000 if rows == 1 else 777) - 1
        c = _case("", "append", batch, rng.randint(1, rows), rows, rng.randint(0, held), held, heads, kv_heads, head_dim, page, kind,
                  qk_norm=rng.random() < 0.3)
    else:
        rows = 1 if op == "decode" else rng.randint(2, 4) if op == "drafts" else _log_int(rng, 5, max(5, min(2048, 4096 // batch)))
        held = _log_int(rng, 1, 8000 if op == "chunk" else 100003) - 1
        c = _case("", "attend", batch, rng.randint(1, rows), rows, rng.randint(0, held), held, heads, kv_heads, head_dim, page, kind,
                  window=rng.choice([0, 0, 0, _log_int(rng, 64, 4096)]), causal=rng.random() < 0.9)
    c.pop("name")
    return c


# ------------------------------------------------------------------ inputs

def _spread(n, lo, hi):
    """n whole numbers from `hi` down to `lo`, evenly over the logarithm."""
    return [hi] if n == 1 else [round(math.exp(math.log(hi + 1) + (math.log(lo + 1) - math.log(hi + 1)) * i / (n - 1))) - 1 for i in range(n)]


def _sizes(case):
    """(held, rows) of each sequence, before the seed's order. The longest prompts are not those of the longest histories."""
    n = case["batch"]
    return _spread(n, case["held_lo"], case["held"]), [max(1, r) for r in reversed(_spread(n, case["rows_lo"], case["rows"]))]


def _rope(positions, head_dim):
    inv = 10000.0 ** (-torch.arange(0, head_dim // 2, dtype=torch.float64, device="cuda") * 2.0 / head_dim)
    ang = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, hq, hkv, d, page = case["batch"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    held, rows = _sizes(case)
    order = torch.randperm(n, device="cuda", generator=g).tolist()
    held, rows = [held[i] for i in order], [rows[i] for i in order]
    need = [-(-(h + r) // page) for h, r in zip(held, rows)]
    pages = sum(need) + 3
    ids = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).tolist()
    table = torch.full((n, max(need) + 1), -1, dtype=torch.int32)      # what a sequence has no page for yet is -1
    for b in range(n):
        table[b, :need[b]] = torch.tensor([ids.pop() for _ in range(need[b])], dtype=torch.int32)
    s = {"op": case["op"], "hq": hq, "hkv": hkv, "d": d, "page": page, "table": table.to("cuda"),
         "lengths": torch.tensor(held, dtype=torch.int32, device="cuda"), "max_rows": case["rows"], "starts": None}
    if case["rows"] > 1:
        s["starts"] = torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32)
    total = sum(rows)
    # keys and values of unit size, pages differing in scale by a factor of up to four; a channel in sixteen stands out, as in
    # the keys of real models
    size = torch.randint(-1, 2, (pages, hkv), device="cuda", generator=g).float()
    stands_out = 1.0 + 2.0 * (torch.rand(hkv, d, device="cuda", generator=g) < 1 / 16)

    def fill():
        x = torch.randn(pages, hkv, page, d, device="cuda", generator=g)
        if case["kind"] == "bf16":
            return (x * stands_out[:, None] * torch.exp2(size)[..., None, None]).to(torch.bfloat16), None
        return (x * stands_out[:, None] * 32).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), torch.exp2(size - 5)

    s["k"], s["k_scale"] = fill()
    s["v"], s["v_scale"] = fill()
    if case["op"] == "append":
        s["qkv"] = torch.randn(total, (hq + 2 * hkv) * d, device="cuda", generator=g).to(torch.bfloat16)
        s["cos"], s["sin"] = _rope(max(held) + case["rows"] + 1, d)
        s["q_gamma"] = s["k_gamma"] = None
        if case["qk_norm"]:
            s["q_gamma"] = 1 + 0.1 * torch.randn(d, device="cuda", generator=g)
            s["k_gamma"] = 1 + 0.1 * torch.randn(d, device="cuda", generator=g)
    else:
        s["q"] = (1.5 * torch.randn(total, hq, d, device="cuda", generator=g)).to(torch.bfloat16)
        s["window"], s["causal"] = case["window"] or None, case["causal"]
    return s


# ------------------------------------------------------------------ the framework's calls and the plain forms

def run(s):
    if own:
        from summa_b200 import ops
        kv = ops.PagedKV(s["k"], s["v"], s["k_scale"], s["v_scale"])
        rows = ops.PagedRows(s["table"], s["lengths"], s["starts"], s["max_rows"])
        if s["op"] == "append":
            q = ops.paged_append(s["qkv"], s["q_gamma"], s["k_gamma"], EPS, s["cos"], s["sin"], s["hq"], s["hkv"], s["d"], kv, rows)
            return _stored(s, q)
        return ops.paged_attention(s["q"], kv, rows, causal=s["causal"], window=s["window"])
    return _append(s) if s["op"] == "append" else _attend(s)


def _stored(s, q):
    """The rotated queries and the whole cache. An 8-bit element stands for its own value times the scale of its page and head, which
    comes along as an output of its own."""
    return {k: v for k, v in {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}.items() if v is not None}


def _places(s, total):
    """Of each row: its sequence, its number there and its position."""
    t = torch.arange(total, device="cuda")
    if s["starts"] is None:
        b, i = t, torch.zeros_like(t)
    else:
        b = (t[:, None] >= s["starts"][None, 1:]).sum(1)
        i = t - s["starts"].long()[b]
    return b, i, s["lengths"].long()[b] + i


def _turn(x, gamma, cos, sin, pos):
    """Norm of each head (with `gamma`), then the rotation of adjacent pairs, in 32 bits."""
    x = x.float()
    if gamma is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma
    c, n = cos[pos][:, None], sin[pos][:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-2)


def _exponent(most):
    """The smallest e with most <= 448 2^e, and no less than -60; in 64 bits, since `most` may lie next to the border."""
    m, e = torch.frexp(most.double() / E4M3_MAX)
    return torch.where(most > 0, torch.where(m > 0.5, e, e - 1), LEAST_EXPONENT).clamp_min(LEAST_EXPONENT)


def _put(pages, scale, x, table, b, pos, lengths):
    """Stores the rows x `[T, Hkv, D]` (32 bits). In 8 bits a page's scale begins anew with its first slot; before that it only grows,
    and what a sequence holds of the page then goes over to the new one."""
    size = pages.shape[2]
    at, slot = table[b, pos // size].long(), pos % size
    if scale is None:
        pages[at, :, slot] = x.to(pages.dtype)
        return
    finite = torch.where(torch.isfinite(x), x.abs(), 0).amax(-1)
    most = torch.full_like(scale, -1.0).index_reduce_(0, at, finite, "amax")
    need = torch.exp2(_exponent(most).double()).float()
    count = lengths.long() % size                                       # what a sequence holds of the page that its first row goes to
    first = table.gather(1, (lengths.long() // size)[:, None])[:, 0].long()
    old = scale[first]
    scale.copy_(torch.where(most >= 0, need, scale))
    scale[first] = new = torch.where(count[:, None] > 0, torch.maximum(old, need[first]), need[first])
    there = pages[first]
    moved = (there.float() * (old / new)[..., None, None]).to(pages.dtype)
    held = torch.arange(size, device="cuda")[:, None] < count[:, None, None, None]
    pages[first] = torch.where(held, moved.float(), there.float()).to(pages.dtype)
    pages[at, :, slot] = torch.where(torch.isfinite(x), x / scale[at][..., None], float("nan")).to(pages.dtype)


def _append(s):
    qkv, hq, hkv, d, page = s["qkv"], s["hq"], s["hkv"], s["d"], s["page"]
    b, _, pos = _places(s, qkv.shape[0])
    x = qkv.unflatten(-1, (-1, d))
    _put(s["k"], s["k_scale"], _turn(x[:, hq:hq + hkv], s["k_gamma"], s["cos"], s["sin"], pos), s["table"], b, pos, s["lengths"])
    _put(s["v"], s["v_scale"], x[:, hq + hkv:].float(), s["table"], b, pos, s["lengths"])
    return _stored(s, _turn(x[:, :hq], s["q_gamma"], s["cos"], s["sin"], pos).to(torch.bfloat16))


def _gathered(pages, scale, table):
    """`[B, Hkv, P * page, D]` in 32 bits."""
    at = table.long().clamp_min(0)
    x = pages[at].float()
    if scale is not None:
        x = x * scale[at][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(s):
    q, hq, hkv, d, n, most = s["q"], s["hq"], s["hkv"], s["d"], s["lengths"].shape[0], s["max_rows"]
    b, i, _ = _places(s, q.shape[0])
    first = s["lengths"].long()
    rows = torch.ones_like(first) if s["starts"] is None else s["starts"].long().diff()
    padded = torch.zeros(n, most, hq, d, device="cuda")
    padded[b, i] = q.float()
    k, v = _gathered(s["k"], s["k_scale"], s["table"]), _gathered(s["v"], s["v_scale"], s["table"])
    x = padded.unflatten(2, (hkv, hq // hkv)).permute(0, 2, 1, 3, 4).flatten(2, 3)              # [B, Hkv, rows * G, D]
    score = torch.matmul(x, k.transpose(-1, -2)).unflatten(2, (most, -1)) * (1 / math.sqrt(d))  # [B, Hkv, rows, G, keys]
    pos = (first[:, None] + torch.arange(most, device="cuda"))[..., None]
    key = torch.arange(k.shape[2], device="cuda")
    seen = key < (first + rows)[:, None, None]
    if s["causal"]:
        seen = seen & (key <= pos)
    if s["window"] is not None:
        seen = seen & ((pos - key).abs() <= s["window"])
    seen = seen[:, None, :, None]
    score = torch.where(seen, score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(score - torch.where(top > float("-inf"), top, 0)), 0)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul((p / torch.where(total > 0, total, 1)).flatten(2, 3), v).unflatten(2, (most, -1))
    return o.permute(0, 2, 1, 3, 4).flatten(2, 3)[b, i].to(q.dtype)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    held, rows = _sizes(case)
    hq, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    size, total = 1 if case["kind"] == "e4m3" else 2, sum(rows)
    if case["op"] == "append":
        positions = min(total, max(h + r for h, r in zip(held, rows)))             # rows of the rotation's table
        return {"bytes": total * ((2 * hq + 2 * hkv) * d * 2 + 2 * hkv * d * size) + positions * d * 4, "flops": total * (hq + hkv) * d * 3}
    pairs = keys = 0
    for h, r in zip(held, rows):
        pos = range(h, h + r)
        w = case["window"] or (h + r)
        hi = [min(p, h + r - 1) if case["causal"] else min(p + w, h + r - 1) for p in pos]
        lo = [max(0, p - w) for p in pos]
        pairs += sum(b - a + 1 for a, b in zip(lo, hi))
        keys += hi[-1] - lo[0] + 1
    return {"bytes": total * hq * d * 4 + keys * 2 * hkv * d * size, "flops": pairs * hq * 4 * d}


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    """Sequence by sequence, one head or page at a time, in 64 bits."""
    s = prepare(case, seed)
    held = s["lengths"].tolist()
    starts = s["starts"].tolist() if s["starts"] is not None else list(range(len(held) + 1))
    return _exact_append(s, held, starts) if s["op"] == "append" else _exact_attend(s, held, starts)


def _exact_append(s, held, starts):
    hq, hkv, d, page = s["hq"], s["hkv"], s["d"], s["page"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    pos = torch.cat([torch.arange(h, h + starts[b + 1] - starts[b], device="cuda") for b, h in enumerate(held)])
    z = torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])[:, None]

    def turned(y, gamma):
        if gamma is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * gamma.double()
        return torch.view_as_real(torch.view_as_complex(y.reshape(*y.shape[:-1], d // 2, 2).contiguous()) * z).reshape(y.shape)

    out = {"q": turned(x[:, :hq], s["q_gamma"])}
    table = s["table"].tolist()
    for name, rows in (("k", turned(x[:, hq:hq + hkv], s["k_gamma"])), ("v", x[:, hq + hkv:])):
        pages, scale = s[name].double(), s[name + "_scale"]
        scale = None if scale is None else scale.double()
        for b, h in enumerate(held):
            end, t = h + starts[b + 1] - starts[b], starts[b]
            while h < end:
                n, at, slot = min(page - h % page, end - h), table[b][h // page], h % page
                new = rows[t:t + n].transpose(0, 1)                                   # [Hkv, n, D]
                if scale is not None:
                    most = new.abs().amax((1, 2))
                    e = torch.ceil(torch.log2(most) - math.log2(E4M3_MAX)).clamp_min(LEAST_EXPONENT)
                    e = torch.where(E4M3_MAX * torch.exp2(e - 1) >= most, e - 1, torch.where(E4M3_MAX * torch.exp2(e) < most, e + 1, e))
                    to = torch.exp2(e.clamp_min(LEAST_EXPONENT))
                    if slot:
                        to = torch.maximum(to, scale[at])
                        pages[at, :, :slot] = _e4m3(pages[at, :, :slot] * (scale[at] / to)[:, None, None])
                    scale[at] = to
                    new = _e4m3(new / to[:, None, None])
                pages[at, :, slot:slot + n] = new
                h, t = h + n, t + n
        out[name] = pages
        if scale is not None:
            out[name + "_scale"] = scale
    return out


def _e4m3(x):
    """To the nearest e4m3 value, ties to even: steps of 2^-3 of the binade, 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_attend(s, held, starts):
    hq, hkv, d, page = s["hq"], s["hkv"], s["d"], s["page"]
    if s["q"].shape[0] * max(held) * hq * s["d"] > 1e12:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, h in enumerate(held):
        r = starts[b + 1] - starts[b]
        ids = s["table"][b, :-(-(h + r) // page)].long()
        pos, key = torch.arange(h, h + r, device="cuda")[:, None], torch.arange(h + r, device="cuda")[None]
        hidden = (key > pos) if s["causal"] else torch.zeros(r, h + r, dtype=torch.bool, device="cuda")
        if s["window"] is not None:
            hidden = hidden | (key > pos + s["window"]) | (key < pos - s["window"])
        for kh in range(hkv):
            k, v = (s[n][ids, kh].double() * (1.0 if s[n + "_scale"] is None else s[n + "_scale"][ids, kh].double()[:, None, None])
                    for n in ("k", "v"))
            k, v = k.reshape(-1, d)[:h + r], v.reshape(-1, d)[:h + r]
            for j in range(kh * (hq // hkv), (kh + 1) * (hq // hkv)):
                score = (s["q"][starts[b]:starts[b] + r, j].double() @ k.t() / d ** 0.5).masked_fill(hidden, float("-inf"))
                out[starts[b]:starts[b] + r, j] = torch.softmax(score, -1) @ v
    return out
