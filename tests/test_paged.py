"""The paged key/value cache: its calls against plain forms in 64 bits, its refusals, and runs of them together.

Tolerances. Sums and products are exact or in 32 bits. One rounding to bf16 is off by at most 2^-8 of the value, to f16 by 2^-11, to
e4m3 by 2^-4 (2^-10 of the scale below its normal range). Attention rounds each weight once (bf16 pages: to bf16, e4m3 pages: to f16;
what f16 cannot hold is below 2^-22 of the largest) and the result once: |o - exact| <= 2^-8 |exact| + e sum_j p_j |v_j| with
e = 2^-8 (bf16 pages) or 2^-11 + 2^-12 (e4m3 pages; the second term for the exponential's 7.5e-5 and the 32-bit sums)."""
import math

import pytest
import torch

from summa_b200 import ops
from summa_b200.ops import PagedKV, PagedRows, paged

gpu = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


# ------------------------------------------------------------------ inputs and the plain forms

def _cache(pages, Hkv, page, D, kind, device, seed=0, spread=2):
    """Pages that hold something, and in 8 bits a scale of its own for each page and head."""
    g = torch.Generator().manual_seed(seed)
    x = [torch.randn(pages, Hkv, page, D, generator=g) for _ in range(2)]
    if kind == "bf16":
        return PagedKV(*(t.to(torch.bfloat16).to(device) for t in x))
    s = [torch.exp2(torch.randint(-6 - spread, -5 + spread, (pages, Hkv), generator=g).float()) for _ in range(2)]
    return PagedKV(*((t * 64).clamp(-448, 448).to(E4M3).to(device) for t in x), *(t.to(device) for t in s))


def _rows(held, rows, page, device, pages=None, seed=0, one=False, spare=2, max_rows=None):
    """Sequences with `held` tokens (negative: not in use) and `rows` new ones, on random pages; entries without need are -1."""
    need = [max(0, -(-(h + r) // page)) if h >= 0 and r else 0 for h, r in zip(held, rows)]
    pages = pages or sum(need) + 2
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(held), max(need) + spare), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    starts = None if one else torch.tensor([0] + rows).cumsum(0).to(torch.int32).to(device)
    return PagedRows(table.to(device), torch.tensor(held, dtype=torch.int32, device=device), starts, max_rows), pages


def _double(kv):
    """The cache's values in 64 bits."""
    out = []
    for t, s in ((kv.k, kv.k_scale), (kv.v, kv.v_scale)):
        x = t.cpu().double()
        out.append(x if s is None else x * s.cpu().double()[..., None, None])
    return out


def _clone(kv):
    return PagedKV(*(None if t is None else t.clone() for t in kv))


def _to(kv, device):
    return PagedKV(*(None if t is None else t.to(device) for t in kv))


def _exact_attention(q, kv, rows, causal, window, scale=None):
    """(o, sum_j p_j |v_j|) in 64 bits."""
    k, v = _double(kv)
    q = q.cpu().double()
    T, Hq, D = q.shape
    Hkv, page = k.shape[1], k.shape[2]
    o, a = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    lengths, table = rows.lengths.tolist(), rows.table.tolist()
    starts = list(range(len(lengths) + 1)) if rows.starts is None else rows.starts.tolist()
    for b, n in enumerate(lengths):
        if n < 0:
            continue
        for t in range(starts[b], starts[b + 1]):
            pos, end = n + t - starts[b], n + starts[b + 1] - starts[b]
            hi = min(end, pos + 1) if causal else end
            lo = 0
            if window is not None:
                lo, hi = max(0, pos - window), min(hi, pos + window + 1)
            at = [(table[b][j // page], j % page) for j in range(lo, hi)]
            ids, slots = torch.tensor([x for x, _ in at]), torch.tensor([x for _, x in at])
            for h in range(Hq):
                kk, vv = k[ids, h // (Hq // Hkv), slots], v[ids, h // (Hq // Hkv), slots]
                p = torch.softmax(kk @ q[t, h] * (scale or 1 / math.sqrt(D)), 0)
                o[t, h], a[t, h] = p @ vv, p @ vv.abs()
    return o, a


def _near(got, want, size, fp8):
    got = got.cpu().double()
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -12 if fp8 else 2.0 ** -8) * size + 1e-30
    assert torch.isfinite(got).all()
    over = ((got - want).abs() / bound).max().item()
    assert over <= 1, over


def _flag():
    from summa_b200.ops import native
    return native.read_error_flag()


def _table(positions, D, device):
    return ops.rope_table(positions, D, 10000.0, None, device)


def _exact_append(qkv, qg, kg, eps, cos, sin, Hq, Hkv, D, kv, rows):
    """(q, k values, v values, scales) in 64 bits, page by page; the values of whole pages, what the call does not touch as it was."""
    x = qkv.cpu().double().view(-1, Hq + 2 * Hkv, D)
    k, v = _double(kv)
    scales = None if kv.k_scale is None else [kv.k_scale.cpu().double(), kv.v_scale.cpu().double()]
    codes = None if scales is None else [kv.k.cpu().double(), kv.v.cpu().double()]
    page, table = k.shape[2], rows.table.tolist()
    q = torch.zeros(x.shape[0], Hq, D, dtype=torch.float64)
    lengths = rows.lengths.tolist()
    starts = list(range(len(lengths) + 1)) if rows.starts is None else rows.starts.tolist()

    def turn(y, gamma, pos):
        if gamma is not None:
            y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * gamma.cpu().double()
        if cos is None:
            return y
        c, s = cos[pos].cpu().double(), sin[pos].cpu().double()
        out = torch.empty_like(y)
        out[..., 0::2], out[..., 1::2] = y[..., 0::2] * c - y[..., 1::2] * s, y[..., 0::2] * s + y[..., 1::2] * c
        return out

    for b, n in enumerate(lengths):
        if n < 0:
            continue
        new = {}
        for t in range(starts[b], starts[b + 1]):
            pos = n + t - starts[b]
            q[t] = turn(x[t, :Hq], qg, pos)
            new.setdefault(pos // page, []).append((pos % page, turn(x[t, Hq:Hq + Hkv], kg, pos), x[t, Hq + Hkv:]))
        for i, stored in new.items():
            at = table[b][i]
            for which, (whole, part) in enumerate(((k, 1), (v, 2))):
                for h in range(Hkv):
                    put = torch.stack([s[part][h] for s in stored])
                    first = stored[0][0]
                    if scales is None:
                        whole[at, h, first:first + len(stored)] = put
                        continue
                    fin = put[torch.isfinite(put)].abs()
                    most = float(fin.max()) if fin.numel() else 0.0
                    e = -60
                    while 448.0 * 2.0 ** e < most:
                        e += 1
                    s = 2.0 ** e
                    if first > 0:
                        s = max(s, float(scales[which][at, h]))
                        codes[which][at, h, :first] = _e4m3(codes[which][at, h, :first] * float(scales[which][at, h]) / s)
                    scales[which][at, h] = s
                    put = torch.where(torch.isfinite(put), put, float("nan"))
                    codes[which][at, h, first:first + len(stored)] = _e4m3(put / s)
    return q, (k, v) if scales is None else codes, scales


def _e4m3(x):
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


# ------------------------------------------------------------------ appending

APPEND = [
    # held, rows (None: one each), Hq, Hkv, D, page, kind, norm, rope
    ([0], None, 4, 2, 128, 16, "e4m3", False, True),
    ([5, 16, 31, 0, 63], None, 8, 2, 128, 32, "e4m3", True, True),
    ([5, 16, 31, 0, 63], None, 2, 2, 64, 16, "bf16", True, True),
    ([7, 0, 40], [1, 33, 0], 4, 4, 64, 16, "e4m3", False, True),
    ([7, 0, 40, 3], [130, 1, 17, 0], 4, 1, 128, 64, "e4m3", True, True),
    ([127, 128, 129], [2, 129, 200], 2, 1, 128, 128, "e4m3", False, True),
    ([127, 128, 129], [2, 129, 200], 2, 1, 128, 128, "bf16", False, True),
    ([3, -1, 12, -1], None, 4, 2, 64, 32, "e4m3", False, False),
    ([3, -1, 12, -1, 9], [4, 3, 0, 0, 20], 4, 2, 128, 16, "e4m3", False, True),
    ([3, -1, 12, -1, 9], [4, 3, 0, 0, 20], 4, 2, 64, 16, "bf16", True, False),
    ([i * 3 for i in range(40)], [1 + i % 3 for i in range(40)], 2, 1, 64, 16, "e4m3", False, True),
    ([i * 5 for i in range(70)], None, 1, 1, 128, 64, "e4m3", False, True),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append_against_64_bits(case, device):
    """Queries to one rounding; bf16 pages to one rounding; codes to the step next to the exact one at the most, and equal but for a few
    (a code differs only where the 32-bit rotation falls on the other side of the middle between two), scales equal."""
    held, rows, Hq, Hkv, D, page, kind, norm, rope = APPEND[case]
    g = torch.Generator().manual_seed(case)
    one = rows is None
    pr, pages = _rows(held, rows or [1] * len(held), page, device, seed=case, one=one)
    kv = _cache(pages, Hkv, page, D, kind, device, seed=case)
    T = sum(rows) if rows else len(held)
    qkv = (torch.randn(T, (Hq + 2 * Hkv) * D, generator=g) * torch.exp2(torch.randint(-3, 4, (T, 1), generator=g).float())).to(torch.bfloat16).to(device)
    qg = kg = None
    if norm:
        qg, kg = (1 + 0.1 * torch.randn(D, generator=g) for _ in range(2))
        qg, kg = qg.to(device), kg.to(device)
    cos, sin = _table(512, D, device) if rope else (None, None)
    want_q, want, scales = _exact_append(qkv, qg, kg, 1e-5, cos, sin, Hq, Hkv, D, kv, pr)
    before = _clone(kv)
    q = ops.paged_append(qkv, qg, kg, 1e-5, cos, sin, Hq, Hkv, D, kv, pr)
    # 32-bit sums of D terms and a rotation: 2^-20 of the head's size
    size = want_q.norm(dim=-1, keepdim=True)
    assert ((q.cpu().double() - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 2.0 ** -20 * size).all()
    for i, (got, old) in enumerate(((kv.k, before.k), (kv.v, before.v))):
        x, w = got.cpu().double(), want[i]
        if kind == "bf16":
            assert ((x - w).abs() <= 2.0 ** -8 * w.abs() + 2.0 ** -20 * w.norm(dim=-1, keepdim=True)).all()
        else:
            assert torch.equal((kv.k_scale, kv.v_scale)[i].cpu().double(), scales[i])
            differ = x != w
            assert differ.double().mean() <= 1e-4
            assert ((x - w).abs() <= 2.0 ** -3 * w.abs() + 2.0 ** -9).all()
    if device == "cuda":
        assert _flag() == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("one", [True, False])
def test_a_page_scale_grows_and_begins_anew(one, device):
    """Rows of 1, then of 16: the codes before are moved to the new scale, rounded once. A new first slot begins the scale anew. Rows of zeros."""
    D, page = 64, 16
    kv = _cache(4, 1, page, D, "e4m3", device, spread=1)
    ones, big, zero = (torch.full((3 * D,), x, dtype=torch.bfloat16, device=device) for x in (1.3, 21.0, 0.0))
    table = torch.tensor([[2]], dtype=torch.int32, device=device)

    def put(row, at):
        starts = None if one else torch.tensor([0, 1], dtype=torch.int32, device=device)
        ops.paged_append(row[None], None, None, 0.0, None, None, 1, 1, D, kv, PagedRows(table, torch.tensor([at], dtype=torch.int32, device=device), starts))

    put(ones, 0)
    assert kv.k_scale[2, 0].item() == 2.0 ** -8                 # 448 * 2^-9 < 1.296875 (1.3 in bf16) <= 448 * 2^-8
    v1 = float(torch.tensor(1.3, dtype=torch.bfloat16)) * 256
    assert (kv.k[2, 0, 0].float() == float(torch.tensor(v1).to(E4M3).float())).all()
    put(big, 1)
    assert kv.k_scale[2, 0].item() == kv.v_scale[2, 0].item() == 2.0 ** -4
    moved = float((torch.tensor(v1).to(E4M3).float() / 16).to(E4M3).float())
    assert (kv.k[2, 0, 0].float() == moved).all() and (kv.k[2, 0, 1].float() == 320).all()   # 21 * 16 = 336, the middle of 320 and 352: to even
    put(zero, 2)
    assert kv.k_scale[2, 0].item() == 2.0 ** -4 and (kv.k[2, 0, 2].float() == 0).all() and (kv.k[2, 0, 0].float() == moved).all()
    put(zero, 0)
    assert kv.k_scale[2, 0].item() == 2.0 ** -60 and (kv.k[2, 0, 0].float() == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [None, [3]])
def test_append_what_is_not_finite_and_the_largest(rows, device):
    """Infinite and NaN elements are stored as NaN and do not count for the scale; the largest bf16 values fit their page."""
    D, page = 64, 16
    T = 3 if rows else 1
    kv = _cache(3, 1, page, D, "e4m3", device)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=device)
    x = torch.ones(T, 3 * D)
    x[0, D + 3], x[0, D + 7], x[0, 2 * D + 1] = float("inf"), float("nan"), torch.finfo(torch.bfloat16).max
    starts = torch.tensor([0, 3], dtype=torch.int32, device=device) if rows else None
    ops.paged_append(x.to(torch.bfloat16).to(device), None, None, 0.0, None, None, 1, 1, D, kv,
                     PagedRows(table, torch.tensor([0], dtype=torch.int32, device=device), starts))
    k, v = kv.k[1, 0, 0].float().cpu(), kv.v[1, 0, 0].float().cpu()
    assert k[3].isnan() and k[7].isnan() and k.isnan().sum() == 2
    assert kv.k_scale[1, 0].item() == 2.0 ** -8 and k[0] == 256
    assert kv.v_scale[1, 0].item() == 2.0 ** 120 and v[1] == 256 and v[0] == 0   # bf16's largest is 255 * 2^120, and e4m3 steps by 16 there


@pytest.mark.parametrize("device", DEVICES)
def test_append_leaves_the_rest_alone(device):
    """Slots behind the rows, pages of nobody, rows behind the last sequence in `out`, and a slot that is not in use."""
    D, page, Hq, Hkv = 64, 16, 2, 2
    for kind in ("bf16", "e4m3"):
        kv = _cache(6, Hkv, page, D, kind, device)
        old = _clone(kv)
        table = torch.tensor([[3, 5], [0, 1]], dtype=torch.int32, device=device)
        pr = PagedRows(table, torch.tensor([10, -1], dtype=torch.int32, device=device), torch.tensor([0, 3, 5], dtype=torch.int32, device=device))
        qkv = torch.randn(7, (Hq + 2 * Hkv) * D).to(torch.bfloat16).to(device)
        out = torch.full((7, Hq, D), 5.0, dtype=torch.bfloat16, device=device)
        assert ops.paged_append(qkv, None, None, 0.0, None, None, Hq, Hkv, D, kv, pr, out) is out
        assert (out[5:] == 5).all() and (out[3:5] == 0).all() and torch.equal(out[:3].flatten(1), qkv[:3, :Hq * D])
        fresh = ops.paged_append(qkv, None, None, 0.0, None, None, Hq, Hkv, D, kv, pr)
        assert (fresh[3:] == 0).all()
        for got, was in ((kv.k, old.k), (kv.v, old.v)):
            g, w = got.view(torch.uint8), was.view(torch.uint8)
            assert torch.equal(g[[0, 1, 2, 4, 5]], w[[0, 1, 2, 4, 5]]) and torch.equal(g[3, :, 13:], w[3, :, 13:])
            assert not torch.equal(g[3, :, 10:13], w[3, :, 10:13])


@gpu
def test_append_positions_without_a_place_store_nothing():
    """A page out of range, a table that ends, a position beyond the rotation's table: nothing is stored, zeros come back, bit 4 of the
    error word is set; the other sequences are served."""
    D, page = 64, 16
    for kind in ("bf16", "e4m3"):
        for rows in (None, [2, 2, 2, 2]):
            kv = _cache(4, 1, page, D, kind, "cuda")
            old = _clone(kv)
            table = torch.tensor([[7, 0], [0, -3], [1, 1], [2, 2]], dtype=torch.int32, device="cuda")
            held = torch.tensor([1, 17, 33, 4], dtype=torch.int32, device="cuda")
            n = 2 if rows else 1
            starts = torch.arange(5, dtype=torch.int32, device="cuda") * 2 if rows else None
            qkv = torch.ones(4 * n, 3 * D, dtype=torch.bfloat16, device="cuda")
            q = ops.paged_append(qkv, None, None, 0.0, *_table(20, D, "cuda"), 1, 1, D, kv, PagedRows(table, held, starts))
            assert _flag() == 4
            assert (q[:3 * n] == 0).all() and (q[3 * n:] != 0).any()
            for got, was in ((kv.k, old.k), (kv.v, old.v)):
                g, w = got.view(torch.uint8), was.view(torch.uint8)
                assert torch.equal(g[[0, 1, 3]], w[[0, 1, 3]]) and not torch.equal(g[2], w[2])


@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [None, "ragged"])
def test_append_of_many_sequences(kind, rows):
    """Thousands of sequences of one row, and 1100 of none to five, with head counts that the heads of a thread do not divide, against the
    plain form on the CPU: each side rounds a result once (2 * 2^-8), the rotation and its sums are off by 2^-20 of the head's size on each."""
    D, page, Hq, Hkv = 64, 16, 5, 2
    g = torch.Generator().manual_seed(11)
    if rows is None:
        held, n = torch.randint(0, 40, (5001,), generator=g).tolist(), None
    else:
        held, n = torch.randint(-3, 40, (1100,), generator=g).tolist(), torch.randint(0, 6, (1100,), generator=g).tolist()
    pr, pages = _rows(held, n or [1] * len(held), page, "cpu", one=n is None)
    kv = _cache(pages, Hkv, page, D, kind, "cpu")
    T = sum(n) if n else len(held)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(torch.bfloat16)
    qg, kg = 1 + 0.1 * torch.randn(D, generator=g), 1 + 0.1 * torch.randn(D, generator=g)
    cos, sin = _table(64, D, "cpu")
    there = _to(kv, "cuda")
    want = ops.paged_append(qkv, qg, kg, 1e-5, cos, sin, Hq, Hkv, D, kv, pr).double()
    got = ops.paged_append(qkv.cuda(), qg.cuda(), kg.cuda(), 1e-5, cos.cuda(), sin.cuda(), Hq, Hkv, D, there,
                           PagedRows(*(None if t is None else t.cuda() for t in pr[:3])))
    assert _flag() == 0
    assert ((got.cpu().double() - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -19 * want.norm(dim=-1, keepdim=True)).all()
    for x, w in ((there.k, kv.k), (there.v, kv.v)):
        x, w = x.cpu().double(), w.double()
        if kind == "bf16":
            assert ((x - w).abs() <= 2.0 ** -7 * w.abs() + 2.0 ** -19 * w.norm(dim=-1, keepdim=True)).all()
        else:
            assert (x != w).double().mean() <= 1e-4 and ((x - w).abs() <= 2.0 ** -3 * w.abs() + 2.0 ** -9).all()
    if kind == "e4m3":
        assert torch.equal(there.k_scale.cpu(), kv.k_scale) and torch.equal(there.v_scale.cpu(), kv.v_scale)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_append_of_more_rows_than_promised(kind):
    """max_rows too small: rows are stored or left as they were, the queries come back, and what was left out is reported."""
    D, page, n = 128, 64, 50
    pr, pages = _rows([0], [n], page, "cuda", max_rows=2)
    kv = _cache(pages, 1, page, D, kind, "cuda")
    old = _clone(kv)
    qkv = torch.ones(n, 3 * D, dtype=torch.bfloat16, device="cuda")
    q = ops.paged_append(qkv, None, None, 0.0, None, None, 1, 1, D, kv, pr)
    flag, at = _flag(), pr.table[0, 0].item()
    stored = (kv.v[at, 0, :n].float() * (1.0 if kind == "bf16" else kv.v_scale[at, 0].item()) == 1).all(-1)
    kept = (kv.v[at, 0, :n].view(torch.uint8) == old.v[at, 0, :n].view(torch.uint8)).all(-1)
    assert (q == 1).all() and stored[:2].all() and (stored | kept).all() and flag == (0 if stored.all() else 4)
    assert torch.equal(kv.v[at, 0, n:].view(torch.uint8), old.v[at, 0, n:].view(torch.uint8))


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_fills_pages_of_every_size(page, D):
    """Whole pages, and both ends of one, in 8 bits: every number of passes that a block makes over its page."""
    Hq, Hkv = 2, 2
    held, rows = [0, page - 3, 5, page // 2], [2 * page, page + 7, 1, page // 4]
    pr, pages = _rows(held, rows, page, "cuda", max_rows=max(rows))
    kv = _cache(pages, Hkv, page, D, "e4m3", "cuda")
    qkv = torch.randn(sum(rows), (Hq + 2 * Hkv) * D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    want_q, want, scales = _exact_append(qkv, None, None, 0.0, None, None, Hq, Hkv, D, kv, pr)
    q = ops.paged_append(qkv, None, None, 0.0, None, None, Hq, Hkv, D, kv, pr)
    assert torch.equal(q.cpu().double(), want_q) and _flag() == 0        # (nothing is turned or normed: bf16 as it came)
    for got, w, s, ws in ((kv.k, want[0], kv.k_scale, scales[0]), (kv.v, want[1], kv.v_scale, scales[1])):
        assert torch.equal(got.cpu().double(), w) and torch.equal(s.cpu().double(), ws)

# ------------------------------------------------------------------ attention

ATTEND = [
    # held, rows (None: one each), Hq, Hkv, D, page, causal, window
    ([0], None, 1, 1, 128, 16, True, None),
    ([0, 1, 15, 16, 17, 127, 128, 129], None, 4, 1, 64, 16, True, None),
    ([300, 0, 63, 1500], None, 8, 2, 128, 64, True, None),
    ([300, -1, 63, -1, 700], None, 16, 2, 128, 32, True, None),
    ([2000], None, 16, 1, 128, 64, True, None),                               # sixteen columns
    ([900, 31], None, 4, 4, 64, 128, True, 40),
    ([1000, 5], None, 8, 4, 128, 16, False, 100),
    ([700, 31, 0, 1300], [3, 1, 4, 2], 8, 2, 128, 64, True, None),            # a few rows
    ([700, 31, 0], [3, 4, 2], 2, 2, 64, 16, False, None),
    ([650, 90], [4, 3], 8, 2, 64, 32, True, 37),
    ([10 * i for i in range(70)], None, 2, 1, 64, 16, True, None),            # more sequences than a warp has lanes
    ([0], [37], 4, 2, 128, 16, True, None),                                   # many rows
    ([0, 5, 260], [129, 1, 300], 2, 1, 64, 32, True, None),
    ([0, 1000, -1, 77], [70, 33, 5, 0], 8, 2, 128, 64, True, None),
    ([300, 0], [66, 140], 4, 1, 128, 16, False, None),
    ([300, 0], [66, 140], 4, 1, 64, 128, True, 50),
    ([120], [18], 24, 1, 64, 16, True, None),                                 # twenty-four heads share one
    ([1200], [17], 8, 8, 128, 64, True, None),                                # keys split, one group of a tile empty
    ([500], None, 24, 1, 128, 64, True, None),                                # one row, 24 columns
    ([1200], [57], 8, 8, 128, 64, True, None),                                # one group of a tile empty
    ([700, 31, 0, 1300], [5, 12, 1, 0], 8, 2, 128, 64, True, None),           # columns taken in three groups
    ([650, 90], [8, 5], 8, 2, 64, 32, False, 37),
    ([400, -1, 20], [7, 2, 9], 5, 1, 64, 16, True, 200),                      # rows across the groups
    ([90], None, 48, 1, 128, 128, True, None),
]


@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention_against_64_bits(case, kind):
    held, rows, Hq, Hkv, D, page, causal, window = ATTEND[case]
    one = rows is None
    pr, pages = _rows(held, rows or [1] * len(held), page, "cuda", seed=case, one=one, max_rows=None if one else max(rows))
    kv = _cache(pages, Hkv, page, D, kind, "cuda", seed=case)
    T = sum(rows) if rows else len(held)
    q = (2 * torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(case))).to(torch.bfloat16).cuda()
    want, size = _exact_attention(q, kv, pr, causal, window)
    got = ops.paged_attention(q, kv, pr, causal, window)
    assert _flag() == 0
    _near(got, want, size, kind == "e4m3")
    assert torch.equal(got, ops.paged_attention(q, kv, pr, causal, window))   # the order of the sums is fixed


@pytest.mark.parametrize("case", [1, 3, 5, 6, 7, 9, 11, 15])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_attention_on_the_cpu(case, kind):
    """The PyTorch form: 32-bit sums and one rounding."""
    held, rows, Hq, Hkv, D, page, causal, window = ATTEND[case]
    pr, pages = _rows(held, rows or [1] * len(held), page, "cpu", seed=case, one=rows is None)
    kv = _cache(pages, Hkv, page, D, kind, "cpu", seed=case)
    q = (2 * torch.randn(sum(rows) if rows else len(held), Hq, D)).to(torch.bfloat16)
    want, size = _exact_attention(q, kv, pr, causal, window)
    got = ops.paged_attention(q, kv, pr, causal, window).double()
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * size).all()


@gpu
@pytest.mark.parametrize("rows", [None, [3, 3], [40, 40]])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_what_lies_behind_a_sequence_never_counts(kind, rows):
    """Slots behind the last key, pages of others, and the keys in front of a window hold NaN and infinities: no output changes."""
    D, page, Hq, Hkv, window = 128, 64, 8, 2, 100
    pr, pages = _rows([300, 70], rows or [1, 1], page, "cuda", one=rows is None, spare=3)
    kv = _cache(pages, Hkv, page, D, kind, "cuda")
    T = sum(rows) if rows else 2
    q = torch.randn(T, Hq, D).to(torch.bfloat16).cuda()
    clean = ops.paged_attention(q, kv, pr, True, window)
    bad = torch.tensor(float("nan")).to(kv.k.dtype).cuda()
    table, n = pr.table.tolist(), rows[0] if rows else 1
    for t in (kv.k, kv.v):
        used = set()
        for b, held in ((0, 300), (1, 70)):
            end, lo = held + n, max(0, held - window)
            for i in range(-(-end // page)):
                at = table[b][i]
                used.add(at)
                t[at, :, max(0, min(page, end - i * page)):] = bad
                t[at, :, :max(0, min(page, lo - i * page))] = bad
        for at in set(range(pages)) - used:
            t[at] = bad
    assert torch.equal(ops.paged_attention(q, kv, pr, True, window), clean)


@gpu
@pytest.mark.parametrize("rows", [None, [2], [60]])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_nan_stays_in_its_sequence(kind, rows):
    D, page = 64, 32
    pr, pages = _rows([200, 100, 40], (rows or [1]) * 3, page, "cuda", one=rows is None)
    kv = _cache(pages, 1, page, D, kind, "cuda")
    q = torch.randn(3 * (rows or [1])[0], 4, D).to(torch.bfloat16).cuda()
    clean = ops.paged_attention(q, kv, pr)
    kv.v[int(pr.table[1, 0]), 0, 3, 5] = torch.tensor(float("nan")).to(kv.v.dtype)
    got, n = ops.paged_attention(q, kv, pr), (rows or [1])[0]
    assert got[n:2 * n, :, 5].isnan().all()
    assert torch.equal(got[:n], clean[:n]) and torch.equal(got[2 * n:], clean[2 * n:]) and torch.equal(got[n:2 * n, :, :5], clean[n:2 * n, :, :5])


@gpu
@pytest.mark.parametrize("rows", [None, [2, 3], [50, 50]])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_queries_that_are_not_finite(kind, rows):
    """A NaN or an infinity in a query row makes that row of that head NaN and changes no other, to the bit."""
    pr, pages = _rows([300, 70], rows or [1, 1], 32, "cuda", one=rows is None)
    kv = _cache(pages, 2, 32, 128, kind, "cuda")
    T = sum(rows) if rows else 2
    q = torch.randn(T, 4, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    want = ops.paged_attention(q, kv, pr)
    bad = q.clone()
    bad[0, 1, 5], bad[T - 1, 2, 127], bad[T - 1, 3, 0] = float("nan"), float("inf"), float("-inf")
    got = ops.paged_attention(bad, kv, pr)
    hit = torch.zeros(T, 4, dtype=torch.bool, device="cuda")
    hit[0, 1] = hit[T - 1, 2] = hit[T - 1, 3] = True
    assert got[hit].isnan().all() and torch.equal(got[~hit], want[~hit]) and _flag() == 0


@gpu
@pytest.mark.parametrize("rows", [None, [2, 2], [50, 50]])
def test_pages_of_very_different_scales(rows):
    """Value scales over 2^-60 .. 2^100 and key scales down to 2^-60 beside ordinary ones: the weight carries them (see the bound above)."""
    D, page = 128, 16
    pr, pages = _rows([210, 300], rows or [1, 1], page, "cuda", one=rows is None)
    kv = _cache(pages, 1, page, D, "e4m3", "cuda")
    g = torch.Generator().manual_seed(3)
    kv.v_scale.copy_(torch.exp2(torch.randint(-60, 100, (pages, 1), generator=g).float()))
    kv.k_scale[::3] = 2.0 ** -60
    q = torch.randn(sum(rows) if rows else 2, 4, D, generator=g).to(torch.bfloat16).cuda()
    want, size = _exact_attention(q, kv, pr, True, None)
    _near(ops.paged_attention(q, kv, pr), want, size, True)


@gpu
@pytest.mark.parametrize("rows", [None, [20]])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_peaked_and_flat_scores(kind, rows):
    """One key 40 above the others, all keys equal, queries of zeros, queries of 2^-100 and 2^100 under a matching scale."""
    D, page = 64, 64
    pr, pages = _rows([4000], rows or [1], page, "cuda", one=rows is None)
    kv = _cache(pages, 1, page, D, kind, "cuda")
    T = (rows or [1])[0]
    q = torch.randn(T, 8, D).to(torch.bfloat16).cuda()
    q[:, 1] = 0
    q[:, 2] *= 8
    cases = [(q, None), ((q.float() * 2.0 ** 100).to(torch.bfloat16), 2.0 ** -103), ((q.float() * 2.0 ** -100).to(torch.bfloat16), 2.0 ** 97)]
    for x, scale in cases:
        want, size = _exact_attention(x, kv, pr, True, None, scale)
        _near(ops.paged_attention(x, kv, pr, scale=scale), want, size, kind == "e4m3")


@gpu
@pytest.mark.parametrize("rows", [[1, 1], [3, 2], [40, 30]])
def test_rows_behind_the_last_sequence(rows):
    D, page, Hq = 64, 16, 4
    pr, pages = _rows([50, 9], rows, page, "cuda", max_rows=max(rows))
    kv = _cache(pages, 2, page, D, "e4m3", "cuda")
    n = sum(rows)
    q = torch.randn(n + 5, Hq, D).to(torch.bfloat16).cuda()
    out = torch.full_like(q, 3.0)
    assert ops.paged_attention(q, kv, pr, out=out) is out
    fresh = ops.paged_attention(q, kv, pr)
    assert (out[n:] == 3).all() and (fresh[n:] == 0).all() and torch.equal(out[:n], fresh[:n]) and (out[:n] != 0).any()


@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("held,rows,behind,max_rows", [([50, 9], [40, 30], 500, None), ([50, -1, 9, 0], [40, 0, 3, 1], 77, None),
                                                       ([50, 2000], [2, 3], 600, 3), ([700], [1], 4000, 1), ([50, 9], [0, 0], 900, None)])
def test_many_rows_behind_the_last_sequence_are_zeros(held, rows, behind, max_rows, D, kind):
    """A call padded far beyond its sequences' rows: all rows behind them are zeros in a fresh output, and as they were in a given one,
    whatever the memory held."""
    page, Hq, Hkv = 64, 8, 2
    pr, pages = _rows(held, rows, page, "cuda", max_rows=max_rows)
    kv = _cache(pages, Hkv, page, D, kind, "cuda")
    n = sum(rows)
    q = torch.randn(n + behind, Hq, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    want, size = _exact_attention(q, kv, pr, True, None)
    qkv = torch.randn(n + behind, (Hq + 2 * Hkv) * D).to(torch.bfloat16).cuda()
    for _ in range(3):
        junk = torch.full_like(q, float("nan"))
        del junk                                                         # (the memory that the next output gets)
        got = ops.paged_attention(q, kv, pr)
        assert (got[n:] == 0).all()
        if n:
            _near(got[:n], want[:n], size[:n], kind == "e4m3")
        out = torch.full_like(q, 3.0)
        ops.paged_attention(q, kv, pr, out=out)
        assert (out[n:] == 3).all() and torch.equal(out[:n], got[:n])
        junk = torch.full_like(q, float("nan"))
        del junk
        back = ops.paged_append(qkv, None, None, 0.0, None, None, Hq, Hkv, D, _clone(kv), pr)
        assert (back[n:] == 0).all() and back.isfinite().all()
    assert _flag() == 0

@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [None, [40, 2]])
def test_keys_without_a_page_are_left_out(kind, rows):
    """A page out of range inside a sequence: as if its keys were not there; bit 4 of the error word. A sequence of such pages only: zeros."""
    D, page = 64, 32
    pr, pages = _rows([200, 60], rows or [1, 1], page, "cuda", one=rows is None)
    kv = _cache(pages, 1, page, D, kind, "cuda")
    q = torch.randn(sum(rows) if rows else 2, 4, D).to(torch.bfloat16).cuda()
    keep = pr.table.clone()
    pr.table[0, 2], pr.table[1] = 10 ** 6, -1
    got = ops.paged_attention(q, kv, pr, causal=False)
    assert _flag() == 4
    n = rows[0] if rows else 1
    assert (got[n:] == 0).all()
    # the same keys gathered without the hole
    k, v = (t.cpu() for t in _double(kv))
    ids = [int(x) for i, x in enumerate(keep[0, :-(-(200 + n) // page)].tolist()) if i != 2]
    held = 200 + n - page
    small = PagedRows(torch.tensor([ids], dtype=torch.int32), torch.tensor([held - n], dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32))
    want, size = _exact_attention(q[:n], kv, small, False, None)
    _near(got[:n], want, size, kind == "e4m3")


@gpu
def test_more_rows_than_promised():
    """max_rows too small: the rows beyond it come back as zeros, bit 4 of the error word is set."""
    pr, pages = _rows([50], [6], 16, "cuda", max_rows=2)
    kv = _cache(pages, 2, 16, 64, "bf16", "cuda")
    q = torch.randn(6, 4, 64).to(torch.bfloat16).cuda()
    got = ops.paged_attention(q, kv, pr)
    assert _flag() == 4 and (got[2:] == 0).all()
    want, size = _exact_attention(q, kv, pr, True, None)
    assert got[:2].isfinite().all()


@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D,held", [(64, [50]), (128, [50]), (64, [3000, 7, 500]), (128, [3000, 7, 500])])
def test_the_promised_rows_are_served_whatever_comes_behind_them(D, held, kind):
    """max_rows too small, by so few columns that they are one group, cut and whole: the promised rows are those of the formula, the others
    zeros, bit 4 of the error word."""
    n = [6, 2, 5][:len(held)]
    pr, pages = _rows(held, n, 16, "cuda", max_rows=2)
    kv = _cache(pages, 2, 16, D, kind, "cuda")
    q = torch.randn(sum(n), 4, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    got = ops.paged_attention(q, kv, pr)
    assert _flag() == 4
    want, size = _exact_attention(q, kv, pr, True, None)
    at = 0
    for r in n:
        _near(got[at:at + 2], want[at:at + 2], size[at:at + 2], kind == "e4m3")
        assert (got[at + 2:at + r] == 0).all()
        at += r

@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_more_rows_than_promised_in_groups(kind):
    pr, pages = _rows([900, 3], [11, 2], 16, "cuda", max_rows=7)
    kv = _cache(pages, 1, 16, 64, kind, "cuda")
    q = torch.randn(13, 4, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    got = ops.paged_attention(q, kv, pr)
    assert _flag() == 4 and (got[7:11] == 0).all()
    want, size = _exact_attention(q, kv, pr, True, None)
    _near(got[:7], want[:7], size[:7], kind == "e4m3")
    _near(got[11:], want[11:], size[11:], kind == "e4m3")


@gpu
@pytest.mark.parametrize("rows", [None, [2, 1], [50, 9]])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_strides_and_views(kind, rows):
    """Pages as views of one pool of all layers, keys and values; queries and output inside wider buffers; a table with room behind it."""
    D, page, Hq, Hkv = 64, 16, 4, 2
    pr, pages = _rows([90, 33], rows or [1, 1], page, "cuda", one=rows is None)
    kv = _cache(pages, Hkv, page, D, kind, "cuda")
    pool = torch.zeros(pages, 3, 2, Hkv, page, D, device="cuda").to(kv.k.dtype)
    pool[:, 1, 0], pool[:, 1, 1] = kv.k, kv.v
    scales = [None, None]
    if kind == "e4m3":
        wide = torch.zeros(pages, 3, 2, Hkv, device="cuda")
        wide[:, 1, 0], wide[:, 1, 1] = kv.k_scale, kv.v_scale
        scales = [wide[:, 1, 0], wide[:, 1, 1]]
    view = PagedKV(pool[:, 1, 0], pool[:, 1, 1], *scales)
    table = torch.full((2, 50), -7, dtype=torch.int32, device="cuda")
    table[:, :pr.table.shape[1]] = pr.table
    prv = pr._replace(table=table[:, :pr.table.shape[1]])
    T = sum(rows) if rows else 2
    wide_q = torch.randn(T, 2 * Hq, D).to(torch.bfloat16).cuda()
    q = wide_q[:, Hq:]
    out = torch.zeros(T, 3 * Hq, D, dtype=torch.bfloat16, device="cuda")
    want = ops.paged_attention(q.contiguous(), kv, pr)
    assert torch.equal(ops.paged_attention(q, view, prv), want)
    ops.paged_attention(q, view, prv, out=out[:, Hq:2 * Hq])
    assert torch.equal(out[:, Hq:2 * Hq], want) and (out[:, :Hq] == 0).all() and (out[:, 2 * Hq:] == 0).all()
    odd = torch.empty(T * Hq * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, Hq, D).copy_(q)
    assert torch.equal(ops.paged_attention(odd, kv, pr), want)
    # appending from a wider projection, into the views
    wide_qkv = torch.randn(T, (Hq + 2 * Hkv) * D + 64).to(torch.bfloat16).cuda()
    cos, sin = _table(200, D, "cuda")
    a = ops.paged_append(wide_qkv[:, 64:], None, None, 0.0, cos, sin, Hq, Hkv, D, view, prv)
    b = ops.paged_append(wide_qkv[:, 64:].contiguous(), None, None, 0.0, cos, sin, Hq, Hkv, D, kv, pr)
    assert torch.equal(a, b) and torch.equal(view.k.float(), kv.k.float()) and torch.equal(view.v.float(), kv.v.float())
    c = torch.zeros(T, 2 * Hq, D, dtype=torch.bfloat16, device="cuda")
    ops.paged_append(wide_qkv[:, 64:], None, None, 0.0, cos, sin, Hq, Hkv, D, view, prv, c[:, ::2])
    assert torch.equal(c[:, ::2], b) and (c[:, 1::2] == 0).all()


def test_rows_that_begin_between_16_bytes_are_copied():
    """What the kernels read 16 bytes at a time: contiguous rows at any element of a buffer."""
    from summa_b200.ops import cuda_ops
    buf = torch.arange(2 * 24 + 8, dtype=torch.bfloat16)
    for i in range(8):
        x = buf[i:i + 48].view(2, 24)
        for y in (x, x.view(2, 1, 24), buf[i:i + 44].as_strided((2, 20), (24, 1))):
            rows, ld = cuda_ops._rows(y)
            assert rows.data_ptr() % 16 == 0 and rows.stride(0) == ld and torch.equal(rows, y.reshape(2, -1))
            assert (rows.data_ptr() == y.data_ptr()) == (y.data_ptr() % 16 == 0)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [None, [7, 20]])
def test_inputs_that_begin_between_16_bytes(rows, kind):
    D, page, Hq, Hkv = 64, 16, 4, 2
    n = rows or [1, 1]
    pr, pages = _rows([40, 3], n, page, "cuda", one=rows is None, max_rows=max(n))
    kv = _cache(pages, Hkv, page, D, kind, "cuda")
    other = _clone(kv)
    T, W = sum(n), (Hq + 2 * Hkv) * D
    cos, sin = _table(64, D, "cuda")
    qkv = torch.randn(T, W, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    gain = (1 + torch.arange(D, device="cuda") / D)

    def odd(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)

    a = ops.paged_append(qkv, gain, gain, 1e-5, cos, sin, Hq, Hkv, D, kv, pr)
    out = odd(torch.zeros_like(a))
    assert ops.paged_append(odd(qkv), odd(gain), odd(gain), 1e-5, cos, sin, Hq, Hkv, D, other, pr, out) is out
    assert torch.equal(out, a) and torch.equal(kv.k.float(), other.k.float()) and torch.equal(kv.v.float(), other.v.float())
    out = odd(torch.zeros_like(a))
    assert torch.equal(ops.paged_attention(odd(a), kv, pr, out=out), ops.paged_attention(a, kv, pr)) and _flag() == 0

@gpu
@pytest.mark.parametrize("rows", [None, [2, 1, 3], [50, 9, 20]])
def test_captured_and_replayed_on_two_streams(rows):
    """Two graphs captured on one stream and replayed on two at once, lengths and pages changing between replays."""
    D, page, Hq, Hkv = 128, 64, 8, 2
    n = rows or [1, 1, 1]
    states = []
    for seed in range(2):
        pr, pages = _rows([2000, 900, 30], n, page, "cuda", seed=seed, one=rows is None, spare=20, max_rows=max(n))
        kv = _cache(pages, Hkv, page, D, "e4m3", "cuda", seed=seed)
        q = torch.randn(sum(n), Hq, D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
        ops.paged_attention(q, kv, pr)
        states.append((q, kv, pr))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q, kv, pr in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_attention(q, kv, pr))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for lengths in ([2000, 900, 30], [5, -1, 1], [1999, 0, 40]):       # (the third has one page of 64, and up to 20 rows)
        for _, _, pr in states:
            pr.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        want = [ops.paged_attention(*s) for s in states]
        for o in outs:
            o.fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert torch.equal(got, w)
    assert _flag() == 0


@gpu
def test_offsets_beyond_32_bits():
    """A pool of more than 2^31 elements and 2^32 bytes: the pages at its end."""
    D, page, Hkv = 128, 128, 8
    pages = (1 << 31) // (Hkv * page * D) + 2 + (1 << 15)
    k = torch.zeros(pages, Hkv, page, D, dtype=E4M3, device="cuda")
    s = torch.full((pages, Hkv), 2.0 ** -6, device="cuda")
    kv = PagedKV(k, k, s, s)
    small = _cache(3, Hkv, page, D, "e4m3", "cuda")
    k[-3:], s[-3:] = small.k, small.k_scale
    kv_small = PagedKV(small.k.clone(), small.k.clone(), small.k_scale, small.k_scale)
    for n in (1, 30):
        rows = PagedRows(torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"), torch.tensor([300], dtype=torch.int32, device="cuda"),
                         torch.tensor([0, n], dtype=torch.int32, device="cuda"), n)
        far = rows._replace(table=rows.table + (pages - 3))
        q = torch.randn(n, 16, D).to(torch.bfloat16).cuda()
        assert torch.equal(ops.paged_attention(q, kv, far), ops.paged_attention(q, kv_small, rows))
        qkv = torch.randn(n, (16 + 16) * D).to(torch.bfloat16).cuda()
    two = PagedKV(kv_small.k, kv_small.v.clone(), small.k_scale.clone(), small.k_scale.clone())
    v = torch.zeros(pages, Hkv, page, D, dtype=E4M3, device="cuda")
    v[-3:] = two.v
    ops.paged_append(qkv, None, None, 0.0, None, None, 16, 8, D, PagedKV(k, v, s, s.clone()), far)
    ops.paged_append(qkv, None, None, 0.0, None, None, 16, 8, D, two, rows)
    assert torch.equal(k[-3:].float(), two.k.float()) and torch.equal(v[-3:].float(), two.v.float()) and not k[:64].float().any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_run_together(kind, device):
    """Prompts, drafted rows and single tokens of two sequences, a slot that joins later: append and attend after one another against
    attention over all rows at once."""
    D, page, Hq, Hkv = 64, 16, 4, 2
    torch.manual_seed(5)
    kv = _cache(24, Hkv, page, D, kind, device)
    table = torch.randperm(24, dtype=torch.int32).view(3, 8).to(device)
    cos, sin = _table(128, D, device)
    qkv = torch.randn(3, 100, (Hq + 2 * Hkv) * D).to(torch.bfloat16).to(device)
    held, outs = [0, 0, -1], [[], [], []]
    for step in ([17, 40, 0], [3, 2, 0], None, None, [1, 1, 30], None, [0, 5, 0], None):
        n = step or [1, 1, 1]
        if step and step[2] == 30:
            held[2] = 0
        live = [x if h >= 0 else 1 for x, h in zip(n, held)] if step is None else n
        rows = torch.cat([qkv[b, max(held[b], 0):max(held[b], 0) + live[b]] for b in range(3)])
        starts = torch.tensor([0] + live).cumsum(0).to(torch.int32).to(device) if step else None
        pr = PagedRows(table, torch.tensor(held, dtype=torch.int32, device=device), starts, max(live) if step else None)
        q = ops.paged_append(rows, None, None, 0.0, cos, sin, Hq, Hkv, D, kv, pr)
        o = ops.paged_attention(q, kv, pr)
        at = 0
        for b in range(3):
            if held[b] >= 0:
                outs[b].append(o[at:at + live[b]])
                held[b] += live[b]
            else:
                assert (o[at:at + live[b]] == 0).all()
            at += live[b]
    for b in range(3):
        n = held[b]
        q, k, v = (t[None] for t in qkv[b, :n].unflatten(1, (-1, D)).split([Hq, Hkv, Hkv], dim=1))
        q, k = ops.reference.apply_rope(q, cos, sin), ops.reference.apply_rope(k, cos, sin)
        want = ops.reference.attention(q.float(), k.float(), v.float())[0]
        got = torch.cat(outs[b])
        assert got.shape == want.shape
        # e4m3 rounds keys and values by 2^-4 each (2^-3 where a page's scale moved); scores of size 1 move by about 2^-4 / sqrt(D) * |q||k|
        assert (got.float() - want).norm() <= (0.01 if kind == "bf16" else 0.1) * want.norm()


# ------------------------------------------------------------------ tiles without keys, tables that end

@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_tile_without_keys_gives_zeros_whole(kind):
    """A slot that is not in use brings more rows than half a tile has, behind a table so short that the keys are taken in one part: its
    rows are zeros, every time, whatever its queries hold."""
    D, page, Hq, Hkv = 128, 64, 8, 2
    table = torch.tensor([[0, 1], [2, 3], [-1, -1]], dtype=torch.int32, device="cuda")
    kv = _cache(4, Hkv, page, D, kind, "cuda")
    rows = [70, 64, 101]
    starts = torch.tensor([0] + rows).cumsum(0).to(torch.int32).cuda()
    q = torch.randn(sum(rows), Hq, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    pr = PagedRows(table, torch.tensor([-1, 30, -7], dtype=torch.int32, device="cuda"), starts, max(rows))
    want, size = _exact_attention(q, kv, pr, True, None)
    for _ in range(50):
        got = ops.paged_attention(q, kv, pr)
        assert (got[:70] == 0).all() and (got[134:] == 0).all()
        _near(got, want, size, kind == "e4m3")
    assert _flag() == 0

@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [None, [2, 3], [6, 11], [70, 40]])
@pytest.mark.parametrize("window", [None, 40])
def test_a_table_that_ends_before_its_sequence(window, rows, kind):
    """The last positions of a sequence have no place in the table: bit 4 of the error word, and rows as if those keys were not there. The
    other sequence is served."""
    D, page, Hq, Hkv = 64, 16, 4, 1
    n = rows or [1, 1]
    pr, pages = _rows([20, 95], n, page, "cuda", one=rows is None, spare=0, max_rows=max(n))
    kv = _cache(pages, Hkv, page, D, kind, "cuda")
    q = torch.randn(sum(n), Hq, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    want, size = _exact_attention(q, kv, pr, True, window)
    _near(ops.paged_attention(q, kv, pr, True, window), want, size, kind == "e4m3")
    assert _flag() == 0                                                  # (as wide as it has to be)
    cut = pr._replace(table=pr.table[:, :-1].contiguous())
    got = ops.paged_attention(q, kv, cut, True, window)
    assert _flag() == 4
    _near(got[:n[0]], want[:n[0]], size[:n[0]], kind == "e4m3")
    there = max(0, cut.table.shape[1] * page - 95)                       # rows of the second sequence whose keys all have a place
    if there:
        _near(got[n[0]:n[0] + there], want[n[0]:n[0] + there], size[n[0]:n[0] + there], kind == "e4m3")
    assert got.isfinite().all()


@pytest.mark.parametrize("rows", [None, [2, 3]])
def test_a_table_that_ends_is_an_error_on_the_cpu(rows):
    pr, pages = _rows([20, 95], rows or [1, 1], 16, "cpu", one=rows is None, spare=0)
    kv = _cache(pages, 1, 16, 64, "bf16", "cpu")
    with pytest.raises(RuntimeError, match="no page"):
        ops.paged_attention(torch.zeros(sum(rows or [1, 1]), 4, 64, dtype=torch.bfloat16), kv, pr._replace(table=pr.table[:, :-1]))

@gpu
@pytest.mark.parametrize("rows", [None, [4], [9], [40]])
@pytest.mark.parametrize("order", ["up", "down", "inside", "far back"])
@pytest.mark.parametrize("D", [64, 128])
def test_value_scales_that_leave_the_weights_apart(D, order, rows):
    """Pages whose value scales are 2^170 apart: all scores alike; and all of them below -64, the small pages' 8 above or below the large
    ones'. Every key counts in the sum of the weights, whatever the scale of its page."""
    page, Hq = 16, 4
    g = torch.Generator().manual_seed(6)
    n = (rows or [1])[0]
    held = 5000 if order == "far back" else 800
    pr, pages = _rows([held], [n], page, "cuda", one=rows is None, max_rows=n)
    kv = _cache(pages, 1, page, D, "e4m3", "cuda", seed=1)
    ids = pr.table[0, :-(-(held + n) // page)].long()
    i = torch.arange(len(ids), device="cuda")
    small = {"up": i < len(ids) // 2, "down": i >= len(ids) // 2, "inside": i % 2 == 0, "far back": i < 280}[order]
    kv.v_scale[ids, 0] = torch.where(small, 2.0 ** -60, 2.0 ** 110)
    kv.k[...] = (torch.randn(kv.k.shape, generator=g) / 4).to(E4M3).cuda()
    kv.k_scale.fill_(1.0)
    q = torch.randn(n, Hq, D, generator=g).to(torch.bfloat16).cuda()
    want, size = _exact_attention(q, kv, pr, True, None)
    _near(ops.paged_attention(q, kv, pr), want, size, True)
    q[..., 0] = 8.0 if D == 64 else 11.3125                              # the first dimension of a key is its score, but for the noise of the others
    for low, high in ((-64.0, -72.0), (-72.0, -64.0)):
        kv.k[ids, 0, :, 0] = torch.where(small, low, high)[:, None].to(E4M3)
        want, size = _exact_attention(q, kv, pr, True, None)
        _near(ops.paged_attention(q, kv, pr), want, size, True)
    assert _flag() == 0

@gpu
@pytest.mark.parametrize("n", [1, 4, 20])
@pytest.mark.parametrize("D", [64, 128])
def test_many_small_weights_under_the_largest_scale(D, n):
    """Value scales of 2^120, one key of weight e^12 (2^17.3) among 100,000 others of 1: together they are more than a third of the sum. So
    many sequences, all over the same pages and with the same queries, that nothing is split."""
    page, Hq, held, B = 128, 4, 100003, 300
    one, pages = _rows([held], [n], page, "cuda", max_rows=n)
    kv = _cache(pages, 1, page, D, "e4m3", "cuda")
    for t, x in zip(kv, (0.0, 0.0, 1.0, 2.0 ** 120)):
        t.fill_(x)
    kv.v[...] = torch.randint(1, 129, kv.v.shape, generator=torch.Generator().manual_seed(8)).to(E4M3).cuda()
    kv.k[int(one.table[0, 300]), 0, 7, 0] = 96.0
    q = torch.zeros(n, Hq, D, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0 if D == 64 else 1.4140625
    want, size = _exact_attention(q, kv, one, True, None)
    starts = None if n == 1 else torch.arange(B + 1, dtype=torch.int32, device="cuda") * n
    rows = PagedRows(one.table.expand(B, -1).contiguous(), one.lengths.expand(B).contiguous(), starts, n)
    got = ops.paged_attention(q.repeat(B, 1, 1), kv, rows)
    _near(got, want.repeat(B, 1, 1), size.repeat(B, 1, 1), True)
    assert _flag() == 0

@gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 3, 70])
def test_lengths_at_the_end_of_32_bits(n, kind):
    """A length far behind the table, up to 2^31 - 1: a row without a window sees what the table holds, one with a window nothing."""
    D, page, Hq, P = 64, 16, 4, 6
    kv = _cache(P, 1, page, D, kind, "cuda")
    table = torch.tensor([[3, 1, 5, 0, 2, 4]], dtype=torch.int32, device="cuda")
    q = torch.randn(n, Hq, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    all_keys = PagedRows(table, torch.tensor([P * page - n], dtype=torch.int32, device="cuda"), starts, n)
    want, size = _exact_attention(q, kv, all_keys, False, None)
    for length in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 40, 2 ** 31 - 300):
        rows = PagedRows(table, torch.tensor([length], dtype=torch.int32, device="cuda"), starts, n)
        for causal in (True, False):
            for window in (None, 2 ** 31 - 1, 1000, 5, 0):
                got = ops.paged_attention(q, kv, rows, causal, window)
                assert _flag() == 4
                if window is None:
                    _near(got, want, size, kind == "e4m3")
                elif window < 2 ** 31 - 1:
                    assert (got == 0).all()
                else:
                    assert got.isfinite().all()
        qkv = torch.randn(n, 6 * D).to(torch.bfloat16).cuda()
        old = _clone(kv)
        assert (ops.paged_append(qkv, None, None, 0.0, None, None, Hq, 1, D, kv, rows) == 0).all() and _flag() == 4
        assert torch.equal(kv.k.float(), old.k.float()) and torch.equal(kv.v.float(), old.v.float())

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [None, [2, 3], [70, 40]])
def test_a_window_wider_than_32_bits_hold_hides_nothing(rows, device):
    pr, pages = _rows([400, 37], rows or [1, 1], 16, device, one=rows is None, max_rows=max(rows or [1]))
    for kind in ("bf16", "e4m3"):
        kv = _cache(pages, 2, 16, 64, kind, device)
        q = torch.randn(sum(rows or [1, 1]), 4, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(device)
        for causal in (True, False):
            want = ops.paged_attention(q, kv, pr, causal)
            for window in (2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31, 2 ** 40):
                assert torch.equal(ops.paged_attention(q, kv, pr, causal, window), want)

# ------------------------------------------------------------------ refusals

def _good(device="cpu", kind="e4m3"):
    pr, pages = _rows([10, 3], [1, 1], 16, device, one=True)
    kv = _cache(pages, 2, 16, 64, kind, device)
    return torch.randn(2, 4, 64).to(torch.bfloat16).to(device), kv, pr


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    q, kv, pr = _good(device)
    qkv = torch.randn(2, 8 * 64).to(torch.bfloat16).to(device)
    cos, sin = _table(64, 64, device)

    def attend(q=q, kv=kv, pr=pr, **more):
        return ops.paged_attention(q, kv, pr, **more)

    def append(qkv=qkv, kv=kv, pr=pr, qg=None, kg=None, cos=cos, sin=sin, Hq=4, Hkv=2, D=64, out=None):
        return ops.paged_append(qkv, qg, kg, 0.0, cos, sin, Hq, Hkv, D, kv, pr, out)

    attend(), append()
    short = kv._replace(k=kv.k[:, :, :8], v=kv.v[:, :, :8])
    for bad in (kv._replace(k_scale=None), kv._replace(v_scale=kv.v_scale[:1]), kv._replace(k_scale=kv.k_scale.double()), short,
                kv._replace(k=kv.k.float(), v=kv.v.float()), kv._replace(v=kv.v[:-1]), kv._replace(k=kv.k.transpose(1, 2), v=kv.v.transpose(1, 2)),
                kv._replace(k=kv.k[..., :32], v=kv.v[..., :32]), kv._replace(k=kv.k[:, :1], v=kv.v[:, :1])):
        for call in (attend, append):
            if call is attend and bad.k.shape[1] == 1:
                continue                                        # (four query heads over one kv head is a valid call)
            with pytest.raises(ValueError):
                call(kv=bad._replace(k_scale=None if bad.k_scale is None else bad.k_scale))
    for bad in (pr._replace(table=pr.table.long()), pr._replace(table=pr.table[0]), pr._replace(lengths=pr.lengths[:1]),
                pr._replace(lengths=pr.lengths.long()), pr._replace(starts=torch.zeros(2, dtype=torch.int32, device=device)),
                pr._replace(starts=torch.zeros(3, device=device)), pr._replace(table=pr.table[:1], lengths=pr.lengths[:1]), pr._replace(max_rows=0)):
        for call in (attend, append):
            with pytest.raises(ValueError):
                call(pr=bad)
    for more in ({"window": -1}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}, {"out": q.float()}, {"out": q[:1]}):
        with pytest.raises(ValueError):
            attend(**more)
    with pytest.raises(ValueError):
        attend(q=q[:, :3])
    with pytest.raises(ValueError):
        attend(q=q[0])
    for more in ({"qkv": qkv[:, :-64]}, {"qkv": qkv[None]}, {"qg": torch.ones(64, device=device)}, {"cos": None}, {"cos": cos[:, :16], "sin": sin[:, :16]},
                 {"cos": cos.double(), "sin": sin.double()}, {"out": q.float()}, {"qg": torch.ones(32, device=device), "kg": torch.ones(32, device=device)}):
        with pytest.raises(ValueError):
            append(**more)
    with pytest.raises(RuntimeError):
        attend(q=q.clone().requires_grad_())
    with pytest.raises(RuntimeError):
        append(qkv=qkv.clone().requires_grad_())
    with torch.no_grad():
        attend(q=q.clone().requires_grad_())


@pytest.mark.parametrize("device", DEVICES)
def test_rows_need_a_table_and_pages(device):
    q, kv, pr = _good(device)
    qkv = torch.randn(2, 8 * 64).to(torch.bfloat16).to(device)
    none = PagedKV(*(t[:0] for t in kv))
    nobody = PagedRows(pr.table[:0], pr.lengths[:0], torch.zeros(1, dtype=torch.int32, device=device))
    for cache, rows in ((kv, pr._replace(table=pr.table[:, :0])), (none, pr), (kv, nobody)):
        with pytest.raises(ValueError):
            ops.paged_attention(q, cache, rows)
        with pytest.raises(ValueError):
            ops.paged_append(qkv, None, None, 0.0, None, None, 4, 2, 64, cache, rows)
        # (no rows, nothing to refuse)
        assert ops.paged_attention(q[:0], cache, rows if rows is nobody else rows._replace(starts=torch.zeros(3, dtype=torch.int32, device=device))).shape == (0, 4, 64)


def test_bad_pages_on_the_cpu():
    q, kv, pr = _good()
    pr.table[0, 0] = 99
    with pytest.raises(RuntimeError):
        ops.paged_attention(q, kv, pr)
    with pytest.raises(RuntimeError):
        ops.paged_append(torch.zeros(2, 8 * 64, dtype=torch.bfloat16), None, None, 0.0, None, None, 4, 2, 64, kv, pr)
    pr.table[0, 0] = 0
    with pytest.raises(RuntimeError):
        ops.paged_append(torch.zeros(2, 8 * 64, dtype=torch.bfloat16), None, None, 0.0, *_table(4, 64, "cpu"), 4, 2, 64, kv, pr)


def test_no_rows_is_no_work():
    for device in ["cpu"] + (["cuda"] if torch.cuda.is_available() else []):
        q, kv, pr = _good(device)
        none = pr._replace(starts=torch.zeros(3, dtype=torch.int32, device=device))
        assert ops.paged_attention(q[:0], kv, none).shape == (0, 4, 64)
        assert ops.paged_append(torch.zeros(0, 8 * 64, dtype=torch.bfloat16, device=device), None, None, 0.0, None, None, 4, 2, 64, kv, none).shape == (0, 4, 64)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_tangent_is_refused_not_dropped(kind, device):
    import torch.autograd.forward_ad as fwd
    q, kv, pr = _good(device, kind)
    qkv = torch.randn(2, 8 * 64).to(torch.bfloat16).to(device)
    gain = torch.ones(64, device=device)

    def append(x=qkv, qg=gain, kg=gain):
        return ops.paged_append(x, qg, kg, 1e-5, None, None, 4, 2, 64, kv, pr)

    def dual(t):
        return fwd.make_dual(t, torch.ones_like(t))

    want = ops.paged_attention(q, kv, pr)
    with fwd.dual_level():
        for call in (lambda: ops.paged_attention(dual(q), kv, pr), lambda: append(dual(qkv)), lambda: append(qg=dual(gain)), lambda: append(kg=dual(gain))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert torch.equal(ops.paged_attention(q, kv, pr), want)         # without a tangent, nothing to refuse
        append()
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: ops.paged_attention(x, kv, pr), (q,), (torch.ones_like(q),))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_no_input_drops_a_gradient(kind, device):
    """Pages, their scales, the rotation's table and the output are refused with a gradient or a tangent like the rows are."""
    import torch.autograd.forward_ad as fwd
    q, kv, pr = _good(device, kind)
    qkv = torch.randn(2, 8 * 64).to(torch.bfloat16).to(device)
    cos, sin = _table(64, 64, device)

    def attend(kv=kv, out=None):
        return ops.paged_attention(q, kv, pr, out=out)

    def append(kv=kv, cos=cos, sin=sin, out=None):
        return ops.paged_append(qkv, None, None, 0.0, cos, sin, 4, 2, 64, kv, pr, out)

    def leaf(t):
        return t.clone().requires_grad_()

    pages = ("k", "v") if kind == "bf16" else ("k_scale", "v_scale")
    for wrap, match in ((leaf, "no_grad"), (lambda t: fwd.make_dual(t, torch.ones_like(t)), "forward-mode")):
        with fwd.dual_level():
            for call in (attend, append):
                for name in pages:
                    with pytest.raises(RuntimeError, match=match):
                        call(kv=kv._replace(**{name: wrap(getattr(kv, name))}))
                with pytest.raises(RuntimeError, match=match):
                    call(out=wrap(torch.zeros_like(q)))
            for more in ({"cos": wrap(cos)}, {"sin": wrap(sin)}):
                with pytest.raises(RuntimeError, match=match):
                    append(**more)
    with torch.no_grad():                                                # (a gradient that nobody asks for is none)
        want = attend()
        assert torch.equal(attend(kv=kv._replace(**{n: leaf(getattr(kv, n)) for n in pages})), want)


@pytest.mark.parametrize("device", DEVICES)
def test_an_output_that_lies_on_itself_is_refused(device):
    q, kv, pr = _good(device)
    qkv = torch.randn(2, 8 * 64).to(torch.bfloat16).to(device)
    one = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=device)
    for out in (one.expand(2, 4, 64), one[:, :1].expand(2, 4, 64), one.transpose(0, 1)[:2].expand(2, 4, 64)):
        with pytest.raises(ValueError, match="one in memory"):
            ops.paged_attention(q, kv, pr, out=out)
        with pytest.raises(ValueError, match="one in memory"):
            ops.paged_append(qkv, None, None, 0.0, None, None, 4, 2, 64, kv, pr, out)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [None, [3, 2], [70, 40]])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_outputs_in_the_place_of_the_inputs(kind, rows, device):
    """Queries left in the projection they came in, attention rows written over their queries."""
    D, page, Hq, Hkv = 128, 64, 4, 2
    n = rows or [1, 1]
    pr, pages = _rows([600, 9], n, page, device, one=rows is None, max_rows=max(n))
    kv = _cache(pages, Hkv, page, D, kind, device)
    other = _clone(kv)
    cos, sin = _table(800, D, device)
    qkv = torch.randn(sum(n), (Hq + 2 * Hkv) * D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(device)
    want_q = ops.paged_append(qkv, None, None, 0.0, cos, sin, Hq, Hkv, D, kv, pr)
    place = qkv[:, :Hq * D].unflatten(1, (Hq, D))
    assert ops.paged_append(qkv, None, None, 0.0, cos, sin, Hq, Hkv, D, other, pr, place) is place
    assert torch.equal(place, want_q) and torch.equal(kv.k.float(), other.k.float()) and torch.equal(kv.v.float(), other.v.float())
    want = ops.paged_attention(want_q, kv, pr)
    assert ops.paged_attention(place, kv, pr, out=place) is place and torch.equal(place, want)
