"""Paged KV cache on the GPU: ssd_paged_append (per-head norms, rotation, rounding to the cache's
type), ssd_paged_read and ssd_paged_attention against plain restatements in 64 bits.

Tolerances, from the arithmetic (eps = 2^-24, the error of one f32 rounding):
* codes of rows written without a norm or rotation, and values read back: none, bit for bit;
* a norm and rotation: the sum of squares is a tree of 4 + 5 additions per lane chunk (at most 16
  roundings), so 1 / sqrt has 8 + 3, the two products 2, the rotation 3 more on |a| + |b|: 16 eps
  of |a| + |b| of the pair;
* attention: a score is a sum over head_dim products, its error at most 2^-19 of
  S = scale * sum |q||k| (32 roundings); weights move by twice the largest score error, and the
  weighted sum and its division add 2^-20: |out - exact| <= (2 * 2^-19 max S + 2^-20) sum w |v|.
"""
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import ssdllm  # noqa: E402
from oracle import oracle as ora  # noqa: E402

DEV = "cuda:0"
EPS = 2.0 ** -24
F16, BF16, Q8, Q4 = ssdllm.F16, ssdllm.BF16, ssdllm.Q8_0, ssdllm.Q4_0
TYPES = [F16, BF16, Q8, Q4]
DIMS = [64, 96, 128, 192, 256]


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return ssdllm.Context(0)


def stands_for(x, wtype):
    """The f32 values that the cache type holds for x (float32 array, last axis the head)."""
    t = torch.from_numpy(np.ascontiguousarray(x))
    if wtype == F16:
        return t.half().float().numpy()
    if wtype == BF16:
        return t.bfloat16().float().numpy()
    raw = ora.quantize(np.ascontiguousarray(x.reshape(1, -1)), wtype)
    return ora.dequantize(raw, wtype, x.size).reshape(x.shape)


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def make_table(rng, lens, page, n_pages, width=None):
    need = [-(-n // page) for n in lens]
    width = width or max(1, max(need))
    ids = rng.permutation(n_pages)[:sum(need)]
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table


def fill(ctx, rng, lens, page, hk, d, wtype, spare=2, width=None, scale=1.0):
    """A cache that holds `lens[i]` positions of sequence i; its table and the held values."""
    n_pages = sum(-(-n // page) for n in lens) + spare
    kv = ssdllm.PagedKvCache(ctx, n_pages, page, hk, d, wtype)
    table = make_table(rng, lens, page, n_pages, width)
    total = sum(lens)
    k = (rng.standard_normal((total, hk, d)) * scale).astype(np.float32)
    v = (rng.standard_normal((total, hk, d)) * np.exp(rng.standard_normal((total, 1, 1)))).astype(np.float32)
    seq = np.repeat(np.arange(len(lens)), lens)
    pos = np.concatenate([np.arange(n) for n in lens]) if total else np.zeros(0)
    if total:
        kv.append(torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV), i32(pos), i32(table),
                  seq=i32(seq))
    ks, vs = (stands_for(x, wtype).astype(np.float64) if total else x for x in (k, v))
    first = np.concatenate([[0], np.cumsum(lens)])
    held = [(ks[a:b], vs[a:b]) for a, b in zip(first[:-1], first[1:])]
    return kv, table, held


def attend(q, k, v, keep=None, scale=None):
    """Exact attention of q [heads][d] over k, v [n][hk][d], and the bound on an f32 result."""
    h, d = q.shape
    hk = k.shape[1] if k.ndim == 3 else 1
    if keep is not None:
        k, v = k[keep], v[keep]
    if len(k) == 0:
        return np.zeros((h, d)), np.zeros((h, d))
    q = q.astype(np.float64).reshape(hk, h // hk, d)
    scale = d ** -0.5 if scale is None else scale
    s = np.einsum("hgd,phd->hgp", q, k) * scale
    big = (np.einsum("hgd,phd->hgp", np.abs(q), np.abs(k)) * scale).max(-1)[..., None]
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    out = np.einsum("hgp,phd->hgd", w, v)
    bound = (2 * 2.0 ** -19 * big + 2.0 ** -20) * np.einsum("hgp,phd->hgd", w, np.abs(v))
    return out.reshape(h, d), bound.reshape(h, d)


def check_attention(got, q, held, lens, window=0, scale=None, seq=None, keep=None):
    got = got.cpu().numpy().astype(np.float64).reshape(q.shape)
    for r in range(q.shape[0]):
        s = r if seq is None else seq[r]
        n = max(0, min(int(lens[r]), len(held[s][0])))
        a = max(0, n - window) if window else 0
        sel = np.arange(a, n) if keep is None else np.array([p for p in range(a, n) if keep(s, p)], int)
        ref, bound = attend(q[r], held[s][0], held[s][1], sel, scale)
        bad = np.abs(got[r] - ref) > bound
        assert not bad.any() and np.isfinite(got[r]).all(), \
            (r, s, n, float(np.abs(got[r] - ref).max()), float(bound.max()), int(bad.sum()))


def run_attention(kv, q, lens, table, seq=None, **more):
    qd = torch.from_numpy(q.reshape(q.shape[0], -1)).to(DEV)
    out = torch.full_like(qd, float("nan"))
    kv.attention(qd, i32(lens), i32(table), out, kv.attention_workspace(),
                 seq=None if seq is None else i32(seq), **more)
    return out


# ------------------------------------------------------------------ write and read back
@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("d", DIMS)
def test_written_rows_read_back_bit_for_bit(ctx, wtype, d):
    rng = np.random.default_rng(d + wtype)
    page, hk, lens = 32, 3, [41, 1, 16, 33]
    kv = ssdllm.PagedKvCache(ctx, 8, page, hk, d, wtype)
    table = make_table(rng, lens, page, 8)
    seq = np.repeat(np.arange(4), lens)
    pos = np.concatenate([np.arange(n) for n in lens])
    n = sum(lens)
    k = rng.standard_normal((n, hk, d)).astype(np.float32)
    v = (rng.standard_normal((n, hk, d)) * 10.0 ** rng.integers(-4, 3, (n, hk, 1))).astype(np.float32)
    k[3] = 0.0                     # a row of zeros
    k[5, 0, :32] = -k[5, 0, 7]     # every magnitude of a block the same
    k[5, 0, 7] *= -1
    v[6, 1, ::2] = 0.0
    order = rng.permutation(n)     # rows of sequences and positions in any order
    kv.append(torch.from_numpy(k[order]).to(DEV), torch.from_numpy(v[order]).to(DEV), i32(pos[order]),
              i32(table), seq=i32(seq[order]))
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        ko = torch.full((n, hk * d), float("nan"), dtype=dt, device=DEV)
        vo = torch.full((n, hk, d), float("nan"), dtype=dt, device=DEV)
        kv.read(i32(pos), i32(table), ko, vo, seq=i32(seq))
        for got, x in ((ko, k), (vo, v)):
            want = torch.from_numpy(stands_for(x, wtype).reshape(n, -1)).to(dt)
            assert torch.equal(got.reshape(n, -1).cpu(), want), dt
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
def test_a_write_touches_its_own_position_only(ctx, wtype):
    rng = np.random.default_rng(7)
    kv, table, held = fill(ctx, rng, [64, 40], 16, 2, 128, wtype)
    row = rng.standard_normal((2, 1, 2, 128)).astype(np.float32)
    kv.append(torch.from_numpy(row[0]).to(DEV), torch.from_numpy(row[1]).to(DEV), i32([21]), i32(table),
              seq=i32([1]))
    for s, n in ((0, 64), (1, 40)):
        ko = torch.empty(n, 256, device=DEV)
        vo = torch.empty(n, 256, device=DEV)
        kv.read(i32(np.arange(n)), i32(table), ko, vo, seq=i32([s] * n))
        want = [x.reshape(n, -1).astype(np.float32).copy() for x in held[s]]
        if s == 1:
            for w, x in zip(want, row):
                w[21] = stands_for(x, wtype).reshape(-1)
        assert np.array_equal(ko.cpu().numpy(), want[0]) and np.array_equal(vo.cpu().numpy(), want[1])


def rotate(x, cs, rd, halves):
    """x [rows][heads][d] in 64 bits, cs [rows][rd/2][2]; also |a| + |b| of each element's pair."""
    y, size = x.copy(), np.abs(x)
    if rd:
        i = np.arange(rd // 2)
        a, b = (i, i + rd // 2) if halves else (2 * i, 2 * i + 1)
        c, s = cs[:, None, :, 0], cs[:, None, :, 1]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
        size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return y, size


@pytest.mark.parametrize("d,h,hk", [(64, 6, 2), (96, 3, 3), (128, 8, 1), (192, 2, 2), (256, 4, 2)])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_norm_and_rotation_of_every_head(ctx, d, h, hk, halves, norm):
    rng = np.random.default_rng(d + h + halves + 2 * norm)
    rows, page = 37, 16
    table = make_table(rng, [80], page, 6)
    kv = ssdllm.PagedKvCache(ctx, 6, page, hk, d, F16)
    x = (rng.standard_normal((rows, (h + 2 * hk) * d)) * np.exp(rng.standard_normal((rows, 1)))).astype(np.float32)
    qw, kw = (1 + 0.2 * rng.standard_normal((2, d))).astype(np.float32)
    xd = torch.from_numpy(x).to(DEV)
    q, k, v = xd[:, :h * d], xd[:, h * d:(h + hk) * d], xd[:, (h + hk) * d:]
    for rd in (0, d, d // 2 // 8 * 8):
        cs, rope = None, None
        if rd:
            rope = torch.empty(80, rd // 2, 2, device=DEV)
            ssdllm.rope_table(ctx, rd, 10000.0, 80, rope)
            cs = rope.cpu().numpy()[43 - rows + 1:44].astype(np.float64)
        pos = np.arange(43 - rows + 1, 44)
        qo = torch.full((rows, h * d), float("nan"), device=DEV)
        kw_ = dict(q_norm=torch.from_numpy(qw).to(DEV), k_norm=torch.from_numpy(kw).to(DEV), eps=1e-6) if norm else {}
        kv.append(k, v, i32(pos), i32(table), seq=i32([0] * rows), q=q, q_out=qo, rope=rope,
                  rope_halves=halves, **kw_)
        ko = torch.empty(rows, hk * d, device=DEV)
        vo = torch.empty(rows, hk * d, device=DEV)
        kv.read(i32(pos), i32(table), ko, vo, seq=i32([0] * rows))
        assert torch.equal(vo.cpu(), v.half().float().cpu())
        for got, part, w, cached in ((qo, x[:, :h * d], qw, False), (ko, x[:, h * d:(h + hk) * d], kw, True)):
            y = part.reshape(rows, -1, d).astype(np.float64)
            if norm:
                y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float32(1e-6)) * w
            want, size = rotate(y, cs, rd, halves)
            tol = 16 * EPS * size
            if cached:  # and one rounding to f16
                tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
            err = np.abs(got.cpu().numpy().reshape(want.shape) - want)
            assert (err <= tol).all(), (rd, cached, float((err - tol).max()))
    kv.free()


def test_rotation_table_and_norms_match_the_single_row_operators(ctx):
    """Adjacent pairs with a table of ssd_rope_table: the bits of ssd_rope; the norm: ssd_rmsnorm's
    formula per head (its sum in another order: 16 eps)."""
    rng = np.random.default_rng(3)
    d, h, pos = 128, 4, 1234
    q = rng.standard_normal((1, h * d)).astype(np.float32)
    rope = torch.empty(pos + 1, d // 2, 2, device=DEV)
    ssdllm.rope_table(ctx, d, 500000.0, pos + 1, rope)
    kv = ssdllm.PagedKvCache(ctx, 1, 2048, h, d, F16)
    qd = torch.from_numpy(q).to(DEV)
    out = torch.empty_like(qd)
    kv.append(qd, qd, i32([pos]), i32([[0]]), q=qd, q_out=out, rope=rope)
    want = qd.clone().reshape(-1)
    ssdllm.rope(ctx, want, d, h, pos, 500000.0)
    assert torch.equal(out.reshape(-1), want)
    w = torch.from_numpy((1 + 0.1 * rng.standard_normal(d)).astype(np.float32)).to(DEV)
    kv.append(qd, qd, i32([pos]), i32([[0]]), q=qd, q_out=out, q_norm=w)
    for i in range(h):
        x = qd[0, i * d:(i + 1) * d].clone()
        ssdllm.rmsnorm(ctx, x, w)
        assert torch.all((out[0, i * d:(i + 1) * d] - x).abs() <= 16 * EPS * x.abs())
    kv.free()


def test_strides_and_alignment(ctx):
    """Rows cut out of wider buffers at odd offsets: the scalar path gives the vector path's bits."""
    rng = np.random.default_rng(5)
    d, h, hk, rows = 128, 4, 2, 9
    x = rng.standard_normal((rows, (h + 2 * hk) * d)).astype(np.float32)
    table = i32([[2, 0]])
    seq, pos = i32([0] * rows), i32(np.arange(10, 10 + rows))
    w = torch.from_numpy((1 + 0.1 * rng.standard_normal(2 * d + 1)).astype(np.float32)).to(DEV)
    rope = torch.empty(64 * d + 1, device=DEV)
    got = []
    for off, extra in ((0, 0), (1, 3)):
        wide = torch.zeros(rows, x.shape[1] + off + extra, device=DEV)
        wide[:, off:off + x.shape[1]] = torch.from_numpy(x).to(DEV)
        xd = wide[:, off:off + x.shape[1]]
        wq = w[:d].clone() if off == 0 else torch.cat([w[:1], w[:d]])[1:]
        table_rope = rope[:64 * d].view(64, d // 2, 2)
        ssdllm.rope_table(ctx, d, 1e4, 64, table_rope)
        kv = ssdllm.PagedKvCache(ctx, 3, 16, hk, d, Q8)
        qo = torch.empty(rows, h * d + off + extra, device=DEV)[:, off:off + h * d]
        kv.append(xd[:, h * d:(h + hk) * d], xd[:, (h + hk) * d:], pos, table, seq=seq, q=xd[:, :h * d],
                  q_out=qo, q_norm=wq, k_norm=wq, rope=table_rope)
        o = torch.empty(2, rows, hk * d + off + extra, device=DEV)[:, :, off:off + hk * d]
        kv.read(pos, table, o[0], o[1], seq=seq)
        att = torch.empty(rows, h * d + off + extra, device=DEV)[:, off:off + h * d]
        kv.attention(qo, pos + 1, table, att, kv.attention_workspace(), seq=seq)
        got.append([t.clone().cpu() for t in (qo, o[0], o[1], att)])
        kv.free()
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_queries_may_be_turned_in_place(ctx):
    rng = np.random.default_rng(6)
    q = torch.from_numpy(rng.standard_normal((5, 512)).astype(np.float32)).to(DEV)
    kv = ssdllm.PagedKvCache(ctx, 5, 16, 4, 128, F16)
    rope = torch.empty(16, 64, 2, device=DEV)
    ssdllm.rope_table(ctx, 128, 1e4, 16, rope)
    args = (q, q, i32([3] * 5), i32(np.arange(5)[:, None]))
    out = torch.empty_like(q)
    kv.append(*args, q=q, q_out=out, rope=rope, rope_halves=True)
    same = q.clone()
    kv.append(*args, q=same, q_out=same, rope=rope, rope_halves=True)
    assert torch.equal(out, same)
    kv.free()


def test_padding_rows_and_positions_without_a_page(ctx):
    rng = np.random.default_rng(8)
    kv, table, held = fill(ctx, rng, [30, 20], 16, 2, 64, Q8, width=3)
    assert ctx.device_status() == 0
    k = torch.from_numpy(rng.standard_normal((2, 128)).astype(np.float32)).to(DEV)
    q, qo = torch.ones(2, 256, device=DEV), torch.full((2, 256), float("nan"), device=DEV)
    kv.append(k, k, i32([-1, 5]), i32(table), seq=i32([0, 1]), q=q, q_out=qo)  # padding: silent
    assert ctx.device_status() == 0
    assert torch.equal(qo[0], torch.zeros(256, device=DEV)) and torch.equal(qo[1], q[1])
    for pos, seq in ((40, 0), (4000000, 0), (3, 2), (3, -1)):  # no page, past the table, no such sequence
        kv.append(k[:1], k[:1], i32([pos]), i32(table), seq=i32([seq]), q=q[:1], q_out=qo[:1])
        assert ctx.device_status() == 3  # SSD_ERR_SHAPE, read once
        assert ctx.device_status() == 0
        assert torch.equal(qo[0], torch.zeros(256, device=DEV))
    bad = table.copy()
    bad[0, 0] = 99  # not a page of the pool
    kv.append(k[:1], k[:1], i32([3]), i32(bad), seq=i32([0]))
    assert ctx.device_status() == 3
    rope = torch.zeros(10, 32, 2, device=DEV)
    kv.append(k[:1], k[:1], i32([10]), i32(table), seq=i32([0]), rope=rope)  # past the rotation table
    assert ctx.device_status() == 3
    ko, vo = torch.full((3, 128), float("nan"), device=DEV), torch.full((3, 128), float("nan"), device=DEV)
    kv.read(i32([10, 40, -1]), i32(table), ko, vo, seq=i32([0, 0, 0]))
    assert np.array_equal(ko[0].cpu().numpy(), held[0][0][10].reshape(-1).astype(np.float32))
    assert not ko[1:].any() and not vo[1:].any()
    kv.free()


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("d,h,hk", [(64, 4, 4), (96, 6, 2), (128, 8, 1), (128, 28, 4), (192, 12, 1),
                                    (256, 32, 2)])
def test_attention_of_ragged_lengths(ctx, wtype, d, h, hk):
    rng = np.random.default_rng(d + h + wtype)
    lens = [1, 0, 2, 15, 16, 17, 31, 64, 100, 700, 33]
    kv, table, held = fill(ctx, rng, lens, 16, hk, d, wtype)
    q = rng.standard_normal((len(lens), h, d)).astype(np.float32) * 2
    out = run_attention(kv, q, lens, table)
    check_attention(out, q, held, lens)
    assert not out[1].any()  # length 0
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("lens", [[1], [5], [3001], [20011], [1200, 2, 1, 9000]])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_few_rows_are_split_over_the_length(ctx, wtype, lens, page):
    rng = np.random.default_rng(sum(lens) + wtype + page)
    kv, table, held = fill(ctx, rng, lens, page, 2, 128, wtype)
    q = rng.standard_normal((len(lens), 16, 128)).astype(np.float32)
    check_attention(run_attention(kv, q, lens, table), q, held, lens)
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("window", [1, 7, 16, 40, 333, 5000])
def test_sliding_window(ctx, wtype, window):
    rng = np.random.default_rng(window)
    lens = [1, 16, 41, 360, 1000]
    kv, table, held = fill(ctx, rng, lens, 32, 2, 64, wtype)
    q = rng.standard_normal((len(lens), 6, 64)).astype(np.float32)
    check_attention(run_attention(kv, q, lens, table, window=window), q, held, lens, window=window)
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
def test_pages_given_back_behind_a_window_and_holes(ctx, wtype):
    """Pages that left the window are -1 in the table; a missing page inside it is left out; a row
    whose pages are all missing gives zeros."""
    rng = np.random.default_rng(9)
    page, lens = 16, [200, 200, 50]
    kv, table, held = fill(ctx, rng, lens, page, 2, 128, wtype)
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    gone = table.copy()
    gone[0, :9] = -1          # positions below 144; window 56 begins there
    gone[1, 4] = 10 ** 6      # not a page
    gone[2] = -1
    keep = lambda s, p: 0 <= gone[s, p // page] < kv.n_pages  # noqa: E731
    out = run_attention(kv, q, lens, gone, window=56)
    check_attention(out, q, held, lens, window=56, keep=keep)
    assert not out[2].any()
    check_attention(run_attention(kv, q, lens, gone), q, held, lens, keep=keep)
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_what_lies_outside_the_length_does_not_matter(ctx, wtype, bad):
    """The last page's other positions, and the positions before a window, hold NaN, infinities or
    the largest numbers."""
    rng = np.random.default_rng(10)
    lens, full = [1, 21, 40, 64], 64
    kv, table, held = fill(ctx, rng, [full] * 4, 32, 2, 128, wtype)
    window = 19
    rows = [(s, p) for s, n in enumerate(lens) for p in range(full) if p >= n or p < n - window]
    x = torch.full((len(rows), 256), bad, device=DEV)
    x[:, ::2] *= -1
    kv.append(x, x, i32([p for _, p in rows]), i32(table), seq=i32([s for s, _ in rows]))
    q = rng.standard_normal((4, 8, 128)).astype(np.float32)
    check_attention(run_attention(kv, q, lens, table, window=window), q, held, lens, window=window)
    kv.free()


def test_nan_inside_stays_in_its_row_and_head(ctx):
    rng = np.random.default_rng(11)
    lens = [100, 90]
    kv, table, held = fill(ctx, rng, lens, 16, 2, 64, F16)
    x = rng.standard_normal((1, 2, 64)).astype(np.float32)
    x[0, 1, 5] = np.nan
    kv.append(torch.from_numpy(x).to(DEV), torch.from_numpy(x).to(DEV), i32([50]), i32(table), seq=i32([0]))
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    out = run_attention(kv, q, lens, table).view(2, 4, 64)
    assert torch.isnan(out[0, 2:]).all() and torch.isfinite(out[0, :2]).all()
    check_attention(out[1:], q[1:], held[1:], lens[1:])
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
def test_rows_of_a_prompt_and_a_shared_prefix(ctx, wtype):
    """Several rows of one sequence (each sees positions up to its own), in any order, beside a
    sequence whose first pages are another's."""
    rng = np.random.default_rng(12)
    page = 16
    kv, table, held = fill(ctx, rng, [70, 50], page, 2, 64, wtype)
    shared = np.vstack([table, table[0]])
    shared[2, 2:4] = table[1, 2:4]  # 32 positions of sequence 0, then positions 32.. of sequence 1
    mixed = tuple(np.concatenate([a[:32], b[32:50]]) for a, b in zip(held[0], held[1]))
    held = held + [mixed]
    seq = np.array([0] * 70 + [2, 1, 2, 2])
    lens = np.array(list(range(1, 71)) + [50, 50, 33, 0])
    order = rng.permutation(len(seq))
    seq, lens = seq[order], lens[order]
    q = rng.standard_normal((len(seq), 8, 64)).astype(np.float32)
    check_attention(run_attention(kv, q, lens, shared, seq=seq), q, held, lens, seq=seq)
    kv.free()


def test_lengths_beyond_the_table_and_unknown_sequences(ctx):
    rng = np.random.default_rng(13)
    kv, table, held = fill(ctx, rng, [64, 64], 32, 2, 64, F16)
    q = rng.standard_normal((4, 4, 64)).astype(np.float32)
    lens, seq = [2 ** 31 - 1, -5, 64, 64], [0, 1, 2, -1]
    out = run_attention(kv, q, lens, table, seq=seq)
    check_attention(out[:1], q[:1], held, [64])
    assert not out[1:].any()
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e9])
def test_sizes_of_queries_keys_and_scale(ctx, wtype, size):
    """Tiny and huge numbers: queries by `size`, the scale by its inverse (so the weights stay)."""
    rng = np.random.default_rng(14)
    lens = [257, 30]
    kv, table, held = fill(ctx, rng, lens, 16, 2, 128, wtype)
    q = (rng.standard_normal((2, 16, 128)) * size).astype(np.float32)
    scale = float(np.float32(0.1 / size))
    out = run_attention(kv, q, lens, table, scale=scale)
    check_attention(out, q, held, lens, scale=scale)
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("small", [2e-4, 50.0])
def test_values_of_any_size(ctx, wtype, small):
    """Value rows whose size changes within a sequence by many binades: the error stays in
    proportion to the weighted sum of their magnitudes."""
    rng = np.random.default_rng(15)
    n = 600
    kv = ssdllm.PagedKvCache(ctx, 40, 16, 1, 64, wtype)
    table = make_table(rng, [n], 16, 40)
    k = rng.standard_normal((n, 1, 64)).astype(np.float32)
    v = (rng.standard_normal((n, 1, 64)) * small).astype(np.float32)
    v[300:] *= 30.0
    v[450:] *= 0.01
    kv.append(torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV), i32(np.arange(n)), i32(table),
              seq=i32([0] * n))
    held = [tuple(stands_for(x, wtype).astype(np.float64) for x in (k, v))]
    q = rng.standard_normal((1, 5, 64)).astype(np.float32)
    check_attention(run_attention(kv, q, [n], table), q, held, [n])
    kv.free()


def test_one_strong_position_far_from_the_rest(ctx):
    """Scores that grow and fall along the sequence, one far above the others in the middle: the
    running maximum moves many times and by much."""
    rng = np.random.default_rng(16)
    n, d = 3000, 64
    for wtype in TYPES:
        kv = ssdllm.PagedKvCache(ctx, 200, 16, 1, d, wtype)
        table = make_table(rng, [n], 16, 200)
        q = rng.standard_normal((1, 4, d)).astype(np.float32)
        k = (rng.standard_normal((n, 1, d)) * 0.3 + q[0, 0] * np.linspace(-3, 3, n)[:, None, None]).astype(np.float32)
        k[1234, 0] = 5 * q[0, 1]
        v = rng.standard_normal((n, 1, d)).astype(np.float32)
        kv.append(torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV), i32(np.arange(n)), i32(table),
                  seq=i32([0] * n))
        held = [tuple(stands_for(x, wtype).astype(np.float64) for x in (k, v))]
        check_attention(run_attention(kv, q, [n], table), q, held, [n])
        kv.free()


def test_many_rows(ctx):
    """More rows than threads of a block or blocks of the GPU, most of them of a token or two."""
    rng = np.random.default_rng(17)
    n_seq, rows = 40, 1500
    lens_all = rng.integers(1, 60, n_seq)
    kv, table, held = fill(ctx, rng, [int(x) for x in lens_all], 16, 2, 64, Q8)
    seq = rng.integers(0, n_seq, rows)
    lens = (rng.random(rows) * (lens_all[seq] + 1)).astype(int)
    lens[::5] = 0
    q = rng.standard_normal((rows, 4, 64)).astype(np.float32)
    check_attention(run_attention(kv, q, lens, table, seq=seq), q, held, lens, seq=seq)
    kv.free()


def test_pool_beyond_32_bit_offsets(ctx):
    """A pool of over 4 GiB, the sequence in its last pages."""
    rng = np.random.default_rng(18)
    page, hk, d = 64, 8, 128
    n_pages = (1 << 32) // (page * hk * d * 2 * 2) + 40
    kv = ssdllm.PagedKvCache(ctx, n_pages, page, hk, d, F16)
    n = 130
    table = np.array([[n_pages - 1, n_pages - 30, n_pages - 7]])
    k, v = rng.standard_normal((2, n, hk, d)).astype(np.float32)
    kv.append(torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV), i32(np.arange(n)), i32(table),
              seq=i32([0] * n))
    held = [tuple(stands_for(x, F16).astype(np.float64) for x in (k, v))]
    q = rng.standard_normal((1, 64, d)).astype(np.float32)
    check_attention(run_attention(kv, q, [n], table), q, held, [n])
    ko, vo = torch.empty(n, hk * d, device=DEV), torch.empty(n, hk * d, device=DEV)
    kv.read(i32(np.arange(n)), i32(table), ko, vo, seq=i32([0] * n))
    assert np.array_equal(vo.cpu().numpy(), held[0][1].reshape(n, -1).astype(np.float32))
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
def test_same_bits_every_time_on_any_stream_and_in_a_graph(ctx, wtype):
    rng = np.random.default_rng(19)
    lens = [5000, 3, 900, 0, 2500]
    kv, table, _ = fill(ctx, rng, lens, 64, 2, 128, wtype)
    q = torch.from_numpy(rng.standard_normal((5, 16 * 128)).astype(np.float32)).to(DEV)
    ln, tb = i32(lens), i32(table)
    work = kv.attention_workspace()
    first = torch.empty_like(q)
    kv.attention(q, ln, tb, first, work)
    assert torch.isfinite(first).all()
    for _ in range(3):
        again = torch.full_like(q, float("nan"))
        kv.attention(q, ln, tb, again, work)
        assert torch.equal(first, again)
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), kv.attention_workspace()
    outs = [torch.full_like(q, float("nan")) for _ in range(8)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):  # two streams at once, each with its own workspace
        if i % 2:
            kv.attention(q, ln, tb, o, work)
        else:
            with torch.cuda.stream(side):
                kv.attention(q, ln, tb, o, other)
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)
    g, out = torch.cuda.CUDAGraph(), torch.full_like(q, float("nan"))
    with torch.cuda.graph(g):
        kv.attention(q, ln, tb, out, work)
    for _ in range(2):
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, out)
    ctx.set_pdl(True)  # programmatic dependent launch of the standalone kernels
    try:
        again = torch.full_like(q, float("nan"))
        kv.attention(q, ln, tb, again, work)
        assert torch.equal(first, again)
    finally:
        ctx.set_pdl(False)
    kv.free()


# ------------------------------------------------------------------ refusals
def status(fn, *args, **kw):
    with pytest.raises(ssdllm.SsdError) as e:
        fn(*args, **kw)
    return e.value.status


def test_creation_refuses(ctx):
    make = ssdllm.PagedKvCache
    assert status(make, ctx, 0, 16, 2, 64, F16) == 1
    assert status(make, ctx, 4, 16, 0, 64, F16) == 1
    for page in (0, 8, 17, 24, 8192, -16):
        assert status(make, ctx, 4, page, 2, 64, F16) == 3
    for d in (0, 32, 80, 100, 512):
        assert status(make, ctx, 4, 16, 2, d, F16) == 3
    for t in (ssdllm.F32, ssdllm.Q4_K, 99):
        assert status(make, ctx, 4, 16, 2, 64, t) == 2
    assert status(make, ctx, 1 << 30, 4096, 64, 256, F16) == 7


def test_calls_refuse_what_does_not_fit(ctx):
    kv = ssdllm.PagedKvCache(ctx, 4, 16, 2, 64, Q8)
    tb = i32([[0, 1], [2, 3]])
    k, q = torch.zeros(2, 128, device=DEV), torch.zeros(2, 256, device=DEV)
    pos, o = i32([0, 1]), torch.zeros(2, 256, device=DEV)
    work = kv.attention_workspace()
    att = lambda **c: kv.attention(**{**dict(q=q, length=pos, table=tb, out=o, workspace=work), **c})  # noqa: E731
    app = lambda **c: kv.append(**{**dict(k=k, v=k, pos=pos, table=tb), **c})  # noqa: E731
    assert status(app, k=k.half()) == 1 and status(app, k=k.cpu()) == 1
    assert status(app, k=torch.zeros(2, 130, device=DEV)) == 1
    assert status(app, k=torch.zeros(2, 256, device=DEV)[:, ::2]) == 1
    assert status(app, v=torch.zeros(3, 128, device=DEV)) == 3
    assert status(app, pos=i32([0])) == 3 and status(app, pos=pos.long()) == 1
    assert status(app, table=i32([[0]])) == 3          # two rows, one sequence, no seq
    assert status(app, table=i32([0, 1])) == 1
    assert status(app, q=torch.zeros(2, 192, device=DEV), q_out=torch.zeros(2, 192, device=DEV)) == 3  # 3 heads, 2 of keys
    assert status(app, k_norm=torch.zeros(32, device=DEV)) == 3
    assert status(app, rope=torch.zeros(4, 64, 2, device=DEV)) == 3   # wider than the head
    assert status(app, rope=torch.zeros(4, 2, 2, device=DEV)) == 3    # 4 dims
    assert status(app, rope=torch.zeros(4, 64, device=DEV)) == 3
    assert status(att, q=torch.zeros(2, 192, device=DEV), out=torch.zeros(2, 192, device=DEV)) == 3
    assert status(att, workspace=work[:8]) == 3
    assert status(att, window=-1) == 1 and status(att, scale=float("nan")) == 1
    assert status(att, scale=-1.0) == 1
    assert status(att, out=torch.zeros(3, 256, device=DEV)) == 3
    assert status(att, table=i32([[0]])) == 3
    assert status(kv.read, pos, tb, k.double(), k.double()) == 1
    assert status(kv.read, pos, tb, k, k.half()) == 1
    assert status(kv.read, i32([1]), tb, k, k) == 3
    # the contiguous cache's calls and this one's do not mix
    plain = ssdllm.KvCache(ctx, 16, 2, 64)
    L = ssdllm.lib()
    v0 = torch.zeros(128, device=DEV)
    assert L.ssd_kv_append(ctx.h, kv.h, v0.data_ptr(), v0.data_ptr(), 0, None) == 8
    assert L.ssd_kv_pointers(kv.h, None, None, None, None) == 8
    assert L.ssd_attention_int8(ctx.h, kv.h, q.data_ptr(), 4, 1, o.data_ptr(), None) == 8
    assert L.ssd_attention_int8_noalloc(ctx.h, kv.h, q.data_ptr(), 4, 1, o.data_ptr(), None) == 8
    assert L.ssd_attention_prefill(ctx.h, kv.h, q.data_ptr(), 1, 256, 0, 4, o.data_ptr(), 256, None) == 8
    h, kv.h = kv.h, plain.h
    assert status(att) == 8 and status(app) == 8 and status(kv.read, pos, tb, k, k) == 8
    kv.h = h
    # no rows: nothing to do
    e = torch.zeros(0, 128, device=DEV)
    kv.append(e, e, i32([]), tb)
    kv.read(i32([]), tb, e, e)
    kv.attention(torch.zeros(0, 256, device=DEV), i32([]), tb, torch.zeros(0, 256, device=DEV), work)
    torch.cuda.synchronize()
    assert ctx.device_status() == 0
    plain.free()
    kv.free()


def test_append_refuses_queries_without_a_place_and_parts_of_heads(ctx):
    kv = ssdllm.PagedKvCache(ctx, 4, 16, 2, 64, Q8)
    k, q = torch.zeros(2, 128, device=DEV), torch.zeros(2, 256, device=DEV)
    app = lambda **c: kv.append(k, k, i32([0, 1]), i32([[0, 1], [2, 3]]), **c)  # noqa: E731
    assert status(app, q=q) == 1 and status(app, q_out=q) == 1
    assert status(app, q=torch.zeros(2, 300, device=DEV), q_out=torch.zeros(2, 256, device=DEV)) == 3
    assert status(app, q=q, q_out=torch.zeros(2, 128, device=DEV)) == 1
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("group", [1, 3, 4, 5, 8])
@pytest.mark.parametrize("length", [5, 300, 9000])
def test_a_nan_in_one_query_is_that_heads_alone(ctx, wtype, group, length):
    """However many warps and blocks share the row: its head is NaN throughout, no other is."""
    d, page = 64, 64
    gen = torch.Generator(device=DEV).manual_seed(length + group)
    kv = ssdllm.PagedKvCache(ctx, length // page + 1, page, 2, d, wtype)
    table = torch.arange(length // page + 1, dtype=torch.int32, device=DEV)[None]
    k = torch.randn(length, 2 * d, generator=gen, device=DEV)
    kv.append(k, k, torch.arange(length, dtype=torch.int32, device=DEV), table, seq=i32([0] * length))
    q = torch.randn(1, 2 * group * d, generator=gen, device=DEV)
    want, out = torch.empty_like(q), torch.empty_like(q)
    work = kv.attention_workspace()
    kv.attention(q, i32([length]), table, want, work)
    assert torch.isfinite(want).all()
    bad = group  # the first head of the second KV head
    q[0, bad * d + 7] = float("nan")
    kv.attention(q, i32([length]), table, out, work)
    got = out.view(-1, d)
    assert torch.isnan(got[bad]).all()
    keep = [h for h in range(2 * group) if h != bad]
    # when the running maximum is raised may change: f32 rounding of values of size 1 to 8
    assert (got[keep] - want.view(-1, d)[keep]).abs().max().item() < 64 * 2.0 ** -24 * 8
    assert ctx.device_status() == 0
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("rows", [20, 70])
def test_lengths_of_a_few_tiles_and_many(ctx, wtype, d, rows):
    """One-token rows beside long ones: units that begin and end inside a warp's share, at its very
    ends, and units of several warps and blocks; each row as on its own, within the rounding of
    another order of sums."""
    rng = np.random.default_rng(rows * d)
    hk, group, page = 2, 4, 32
    lens = [int(x) for x in rng.choice([0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 100, 700, 2500], rows)]
    kv = ssdllm.PagedKvCache(ctx, sum(n // page + 1 for n in lens), page, hk, d, wtype)
    table = i32(make_table(rng, lens, page, sum(n // page + 1 for n in lens)))
    gen = torch.Generator(device=DEV).manual_seed(d)
    for r, n in enumerate(lens):
        if n:
            k, v = (torch.randn(n, hk * d, generator=gen, device=DEV) for _ in range(2))
            kv.append(k, v, i32(range(n)), table, seq=i32([r] * n))
    q = torch.randn(rows, hk * group * d, generator=gen, device=DEV)
    out, one = torch.full_like(q, float("nan")), torch.full_like(q, float("nan"))
    work = kv.attention_workspace()
    kv.attention(q, i32(lens), table, out, work)
    for r in range(rows):
        kv.attention(q[r:r + 1], i32(lens[r:r + 1]), table, one[r:r + 1], work, seq=i32([r]))
    # sums of up to 2500 terms in other orders, of values of size 1: 2^-24 a step, tens of steps
    assert (out - one).abs().max().item() < 64 * 2.0 ** -24 * 8
    for r, n in enumerate(lens):
        if n == 0:
            assert (out[r] == 0).all()
    again = torch.empty_like(out)
    kv.attention(q, i32(lens), table, again, work)
    assert torch.equal(again, out)
    assert ctx.device_status() == 0
    kv.free()


# ------------------------------------------------------------------ rows in runs
@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("n,start", [(1, 0), (15, 1), (16, 0), (16, 9), (17, 16), (33, 5), (70, 31)])
def test_runs_of_positions_at_any_start(ctx, wtype, d, n, start):
    """Consecutive positions of one sequence that begin and end inside groups and pages, more KV
    heads than a block takes at once: written and read as runs, the bits of rows on their own."""
    rng = np.random.default_rng(n * 100 + start + d)
    hk, page, last = 9, 16, 112
    kv = [ssdllm.PagedKvCache(ctx, 9, page, hk, d, wtype) for _ in range(2)]
    table = i32(make_table(rng, [last], page, 9))
    old = torch.from_numpy(rng.standard_normal((last, hk * d)).astype(np.float32)).to(DEV)
    k, v = (torch.from_numpy(rng.standard_normal((n, hk * d)).astype(np.float32)).to(DEV) for _ in range(2))
    pos = np.arange(start, start + n)
    for c in kv:
        c.append(old, old, i32(np.arange(last)), table, seq=i32([0] * last))
    kv[0].append(k, v, i32(pos), table, seq=i32([0] * n))
    order = rng.permutation(n)
    if n > 1 and (order == np.arange(n)).all():
        order = order[::-1].copy()
    kv[1].append(k[order], v[order], i32(pos[order]), table, seq=i32([0] * n))
    got = []
    back = rng.permutation(last)
    for c in kv:
        for dt in (torch.float32, torch.bfloat16):
            for rows in (np.arange(last), back):
                o = torch.full((2, last, hk * d), float("nan"), dtype=dt, device=DEV)
                c.read(i32(rows), table, o[0], o[1], seq=i32([0] * last))
                got.append(o[:, torch.from_numpy(np.argsort(rows)).to(DEV)].float().cpu())
            part = torch.full((2, n, hk * d), float("nan"), dtype=dt, device=DEV)
            c.read(i32(pos), table, part[0], part[1], seq=i32([0] * n))
            assert torch.equal(part.float().cpu(), got[-1][:, start:start + n])
    for i in (1, 4, 5):
        assert torch.equal(got[0], got[i])
    for i in (3, 6, 7):
        assert torch.equal(got[2], got[i])
    want = [stands_for(old.cpu().numpy().reshape(last, hk, d), wtype).reshape(last, -1).copy() for _ in range(2)]
    for w, x in zip(want, (k, v)):
        w[start:start + n] = stands_for(x.cpu().numpy().reshape(n, hk, d), wtype).reshape(n, -1)

    assert np.array_equal(got[0].numpy(), np.stack(want))
    for c in kv:
        c.free()


def test_a_run_that_leaves_its_pages_or_the_rotation_table(ctx):
    """A run whose later positions have no page, or no row in the table of rotations: the first ones
    are written, the status says that others were not."""
    rng = np.random.default_rng(21)
    kv = ssdllm.PagedKvCache(ctx, 3, 16, 2, 64, Q8)
    table = i32([[1, 2, -1]])
    x = torch.from_numpy(rng.standard_normal((16, 128)).astype(np.float32)).to(DEV)
    zero = torch.zeros(48, 128, device=DEV)
    for start, rope, last in ((24, None, 32), (10, torch.ones(20, 32, 2, device=DEV), 20)):
        kv.append(zero[:32], zero[:32], i32(np.arange(32)), table, seq=i32([0] * 32))
        assert ctx.device_status() == 0
        kv.append(x, x, i32(np.arange(start, start + 16)), table, seq=i32([0] * 16), rope=rope)
        assert ctx.device_status() == 3
        ko, vo = torch.full((48, 128), float("nan"), device=DEV), torch.full((48, 128), float("nan"), device=DEV)
        kv.read(i32(np.arange(48)), table, ko, vo, seq=i32([0] * 48))
        want = torch.zeros(48, 128)
        want[start:last] = torch.from_numpy(stands_for(x.cpu().numpy(), Q8))[:last - start]
        assert torch.equal(vo.cpu(), want)
        assert not ko[last:].any() and not ko[:start].any() and ko[start:last].any()
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("turned", [False, True])
def test_positions_up_to_the_largest_number(ctx, wtype, turned):
    """The table's last position, the first one behind it and the largest numbers there are, alone
    and as runs of 16: what has no page is reported, writes nothing and reads as zeros."""
    rng = np.random.default_rng(22)
    page, hk, d, cap, top = 16, 2, 64, 48, 2 ** 31 - 1
    kv = ssdllm.PagedKvCache(ctx, 3, page, hk, d, wtype)
    table = i32([[2, 0, 1]])
    rope = torch.tensor([1.0, 0.0], device=DEV).repeat(64, d // 2, 1) if turned else None
    zero = torch.zeros(cap, hk * d, device=DEV)
    x = torch.from_numpy(rng.standard_normal((16, hk * d)).astype(np.float32)).to(DEV)
    held = torch.from_numpy(stands_for(x.cpu().numpy(), wtype))
    for first, n in ((cap - 1, 1), (cap, 1), (cap - 16, 16), (cap - 8, 16), (cap, 16), (top - 31, 16), (top - 16, 1),
                     (top - 15, 1), (top - 15, 16), (top - 7, 4), (top - 1, 2), (top - 1, 1), (top, 1)):
        kv.append(zero, zero, i32(np.arange(cap)), table, seq=i32([0] * cap))
        pos, seq = i32(np.arange(first, first + n)), i32([0] * n)
        qo = torch.full((n, 2 * hk * d), float("nan"), device=DEV)
        kv.append(x[:n], x[:n], pos, table, seq=seq, q=torch.ones_like(qo), q_out=qo, rope=rope, rope_halves=True)
        kept = max(0, min(n, cap - first))
        assert ctx.device_status() == (0 if kept == n else 3)
        assert (qo[:kept] == 1).all() and (qo[kept:] == 0).all()
        whole = torch.zeros(cap, hk * d)
        whole[first:first + kept] = held[:kept]
        part = torch.cat([held[:kept], torch.zeros(n - kept, hk * d)])
        for at, want in ((np.arange(cap), whole), (np.arange(first, first + n), part)):
            o = torch.full((2, len(at), hk * d), float("nan"), device=DEV)
            kv.read(i32(at), table, o[0], o[1], seq=i32([0] * len(at)))
            assert torch.equal(o[0].cpu(), want) and torch.equal(o[1].cpu(), want), (first, n)
    kv.free()


@pytest.mark.parametrize("d", [64, 256])
def test_the_last_pages_of_the_longest_table(ctx, d):
    """A table of 2^27 - 1 pages of 16 positions, as long as one may be: its last positions."""
    rng = np.random.default_rng(23)
    pages, n = 2 ** 27 - 1, 41
    end = pages * 16
    kv = ssdllm.PagedKvCache(ctx, 4, 16, 1, d, F16)
    table = torch.full((1, pages), -1, dtype=torch.int32, device=DEV)
    table[0, -3:] = i32([3, 0, 2])
    k, v = rng.standard_normal((2, n, 1, d)).astype(np.float32)
    pos = torch.arange(end - n, end, device=DEV).to(torch.int32)
    seq = i32([0] * n)
    kv.append(torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV), pos, table, seq=seq)
    assert ctx.device_status() == 0
    held = [tuple(stands_for(x, F16).astype(np.float64) for x in (k, v))]
    o = torch.full((2, n, d), float("nan"), device=DEV)
    kv.read(pos, table, o[0], o[1], seq=seq)
    for got, want in zip(o, held[0]):
        assert np.array_equal(got.cpu().numpy(), want.reshape(n, d).astype(np.float32))
    q = rng.standard_normal((1, 4, d)).astype(np.float32)
    out = torch.full((1, 4 * d), float("nan"), device=DEV)
    for window in (1, 30, n):
        kv.attention(torch.from_numpy(q.reshape(1, -1)).to(DEV), torch.tensor([end], device=DEV).to(torch.int32), table,
                     out, kv.attention_workspace(), window=window)
        check_attention(out, q, held, [n], window=window)
    assert ctx.device_status() == 0
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("size", [1e6, 1e8, 1e10, 1e20, 1e34])
@pytest.mark.parametrize("n", [30, 300, 9000])
def test_large_scores(ctx, wtype, size, n):
    """Scores far beyond what an f32 number holds to a whole unit: the largest has all the weight;
    equal ones, positive or negative, share it."""
    rng = np.random.default_rng(25)
    d, h, hk, at = 64, 8, 2, n - 7
    q = ((0.5 + rng.random((1, h, d))) * size).astype(np.float32)
    v = rng.standard_normal((n, hk, d)).astype(np.float32)
    vs = stands_for(v, wtype).astype(np.float64)
    for kind in ("one", "equal", "equal and negative"):
        k = np.repeat(rng.random((1, hk, d)) + 0.5, n, 0).astype(np.float32) * (-1 if "neg" in kind else 1)
        if kind == "one":
            k[:] = rng.standard_normal((n, hk, d)) * 0.05
            k[at] = 1.0
        kv = ssdllm.PagedKvCache(ctx, n // 32 + 1, 32, hk, d, wtype)
        table = make_table(rng, [n], 32, n // 32 + 1)
        kv.append(torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV), i32(np.arange(n)), i32(table),
                  seq=i32([0] * n))
        if kind == "one":
            s = np.einsum("hgd,phd->hgp", q[0].astype(np.float64).reshape(hk, h // hk, d), stands_for(k, wtype)) / 8
            assert (s[..., at, None] - np.delete(s, at, -1) > 0.3 * 8 * size).all()  # e^-margin is nothing
            want = vs[at]
            bound = 2.0 ** -20 * np.abs(want)
        else:
            want, bound = vs.mean(0), 2.0 ** -20 * np.abs(vs).mean(0)
        got = run_attention(kv, q, [n], table).cpu().numpy().astype(np.float64).reshape(hk, h // hk, d)
        assert (np.abs(got - want[:, None]) <= bound[:, None]).all(), kind
        kv.free()


@pytest.mark.parametrize("d,h,hk", [(64, 8, 2), (128, 16, 2), (256, 6, 1)])
@pytest.mark.parametrize("key,size", [(1e33, 1.0), (1e36, 1.0), (3e38, 1e-3), (3e38, 1e-30), (1e-6, 1e30), (1.0, 1e36)])
def test_largest_keys_of_a_bf16_cache(ctx, d, h, hk, key, size):
    """Keys and queries of any size whose scores are f32 numbers: a position far above the others
    has all the weight, one far below them none."""
    rng = np.random.default_rng(24)
    n, at, scale = 300, 211, 0.1
    q = ((0.5 + rng.random((1, h, d))) * size).astype(np.float32)
    k = (rng.standard_normal((n, hk, d)) * min(1.0, 1.0 / size)).astype(np.float32)
    v = rng.standard_normal((n, hk, d)).astype(np.float32)
    for sign in (1.0, -1.0):
        kv = ssdllm.PagedKvCache(ctx, 20, 16, hk, d, BF16)
        table = make_table(rng, [n], 16, 20)
        k[at] = sign * key
        kv.append(torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV), i32(np.arange(n)), i32(table),
                  seq=i32([0] * n))
        ks, vs = (stands_for(x, BF16).astype(np.float64) for x in (k, v))
        s = np.einsum("hgd,phd->hgp", q[0].astype(np.float64).reshape(hk, h // hk, d), ks) * scale
        margin = sign * (s[..., at, None] - np.delete(s, at, -1))
        assert (margin > 1e6).all()  # e^-margin is nothing, whatever the rounding of the scores
        want, bound = attend(q[0], ks, vs, np.array([at]) if sign > 0 else np.delete(np.arange(n), at), scale)
        if sign > 0:
            bound = 2.0 ** -20 * np.abs(want)
        got = run_attention(kv, q, [n], table, scale=scale).cpu().numpy().astype(np.float64).reshape(h, d)
        assert (np.abs(got - want) <= bound).all()
        kv.free()


@pytest.mark.parametrize("n", [40, 300, 9000])
@pytest.mark.parametrize("size", [1e-20, 1e33, 1e36, 3e38])
def test_largest_values_of_a_bf16_cache(ctx, n, size):
    """Values near the largest number there is, under scores that rise along the sequence (the running
    maximum lags behind): their average is a number as well, if their sum is one."""
    rng = np.random.default_rng(26)
    d, h, hk = 64, 8, 2
    size = min(size, 3e37) if n == 9000 else size  # some 600 of them count
    kv = ssdllm.PagedKvCache(ctx, n // 32 + 1, 32, hk, d, BF16)
    table = make_table(rng, [n], 32, n // 32 + 1)
    q = (rng.random((1, h, d)) + 0.5).astype(np.float32)
    k = (0.02 * rng.standard_normal((n, hk, d)) + np.linspace(0, 1.4, n)[:, None, None]).astype(np.float32)
    v = ((1 - 0.5 * rng.random((n, hk, d))) * rng.choice([-size, size], (1, hk, d))).astype(np.float32)
    kv.append(torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV), i32(np.arange(n)), i32(table),
              seq=i32([0] * n))
    held = [tuple(stands_for(x, BF16).astype(np.float64) for x in (k, v))]
    check_attention(run_attention(kv, q, [n], table), q, held, [n])
    kv.free()


@pytest.mark.parametrize("nats", [25, 60, 75])
@pytest.mark.parametrize("d,group", [(64, 3), (128, 8), (256, 5)])
def test_small_weights_beside_a_bf16_cache(ctx, nats, d, group):
    """A position with values of zero, its score far above all others': their weights count, however
    small."""
    rng = np.random.default_rng(30)
    n, hk = 200, 2
    kv = ssdllm.PagedKvCache(ctx, 8, 32, hk, d, BF16)
    table = make_table(rng, [n], 32, 8)
    q = (rng.random((1, group * hk, d)) + 0.5).astype(np.float32)
    k = (0.002 * rng.standard_normal((n, hk, d))).astype(np.float32)
    v = rng.standard_normal((n, hk, d)).astype(np.float32)
    k[70], v[70] = nats / d ** 0.5, 0.0
    kv.append(torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV), i32(np.arange(n)), i32(table),
              seq=i32([0] * n))
    held = [tuple(stands_for(x, BF16).astype(np.float64) for x in (k, v))]
    check_attention(run_attention(kv, q, [n], table), q, held, [n])
    kv.free()


def hold(ctx, rng, k, v, page, wtype):
    """A cache that holds k and v of one sequence; its table and the held values."""
    n, hk, d = k.shape
    pages = n // page + 2
    kv = ssdllm.PagedKvCache(ctx, pages, page, hk, d, wtype)
    table = make_table(rng, [n], page, pages)
    k, v = k.astype(np.float32), v.astype(np.float32)
    kv.append(torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV), i32(np.arange(n)), i32(table),
              seq=i32([0] * n))
    return kv, table, [tuple(stands_for(x, wtype).astype(np.float64) for x in (k, v))]


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("nats", [8, 14, 17, 25, 40, 75])
@pytest.mark.parametrize("d,group", [(64, 3), (128, 8), (256, 5)])
def test_a_strong_position_with_zero_values(ctx, wtype, nats, d, group):
    """One position's score is far above the others' and its V is zero: what counts are weights far
    below the largest, alone and beside values 2^8 to 2^20 times as large of positions with no weight
    to speak of, of other blocks of dims, or of the same tile's positions."""
    rng = np.random.default_rng(27)
    n, hk = 200, 2
    q = (rng.random((1, group * hk, d)) + 0.5).astype(np.float32)
    k1 = 0.002 * rng.standard_normal((n, hk, d))
    k1[70] = nats / (d * d ** -0.5)
    v1 = rng.standard_normal((n, hk, d))
    v1[70] = 0.0
    for shape in ("equal", "before", "blocks", "ragged"):
        for size in (2.0 ** 8, 2.0 ** 12, 2.0 ** 20):
            k, v = k1.copy(), v1.copy()
            if size > 2.0 ** 15:
                v *= 2.0 ** -8  # f16 ends at 2^16
            if shape == "before":     # tiles before it and its own
                k[[3, 66]] = -60 / (d * d ** -0.5)
                v[[3, 66]] *= size
            elif shape == "blocks":   # dims 32 to 63
                v[:, :, 32:64] *= size
            elif shape == "ragged":   # every other position
                k[::2] += -20 / (d * d ** -0.5)
                v[::2] *= size
                v[70] = 0.0
            kv, table, held = hold(ctx, rng, k, v, 32, wtype)
            check_attention(run_attention(kv, q, [n], table), q, held, [n])
            check_attention(run_attention(kv, q, [75], table, window=30), q, held, [75], window=30)
            kv.free()
            if shape == "equal":
                break


@pytest.mark.parametrize("wtype", [Q8, Q4])
@pytest.mark.parametrize("top", [2.0 ** 18, 1.0, 2.0 ** -10])
@pytest.mark.parametrize("nats", [0, 5, 30])
def test_value_scales_of_every_size(ctx, wtype, top, nats):
    """V whose blocks' scales go through all of f16's range and are zero, under equal and very different
    weights: every block's output is in proportion to what is in that block."""
    rng = np.random.default_rng(28)
    n, hk, h, d = 333, 1, 4, 256
    q = (rng.random((1, h, d)) + 0.5).astype(np.float32)
    k = 0.002 * rng.standard_normal((n, hk, d)) - np.linspace(0, nats, n)[:, None, None] / (d * d ** -0.5)
    top = min(top, 2.0 ** 15) if wtype == Q4 else top  # a scale is the largest value's eighth, and an f16 number
    v = rng.standard_normal((n, hk, d)) * top * np.repeat(2.0 ** -np.arange(0, 32, 4), 32)
    v[100:200] = 0.0
    v[:, :, 64:96] *= 2.0 ** -rng.integers(0, 12, (n, 1, 1))
    kv, table, held = hold(ctx, rng, k, v, 16, wtype)
    check_attention(run_attention(kv, q, [n], table), q, held, [n])
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_nan_and_infinite_values_beside_small_weights(ctx, wtype, bad):
    """A V that is not a number makes its block's outputs so, not others', when weights need passes of
    their own; outside the range it does not matter."""
    rng = np.random.default_rng(29)
    n, d = 90, 64
    q = (rng.random((1, 4, d)) + 0.5).astype(np.float32)
    k = 0.002 * rng.standard_normal((n, 1, d))
    k[40] = 30 / 8
    v = rng.standard_normal((n, 1, d)) * np.repeat([1.0, 2.0 ** 12], 32)
    v[60:, :, :32] = 3e38 if wtype != F16 and wtype != BF16 and bad > 0 else bad  # 8- and 4-bit codes of NaN are numbers
    if wtype in (Q8, Q4) and bad != bad:
        v[60:, :, :32] = np.inf
    with np.errstate(all="ignore"):
        kv, table, held = hold(ctx, rng, k, v, 16, wtype)
        out = run_attention(kv, q, [60], table).view(4, d)
        check_attention(out[None], q, [(held[0][0][:60], held[0][1][:60])], [60])
        out = run_attention(kv, q, [n], table).cpu().numpy().astype(np.float64).reshape(4, d)
        assert not np.isfinite(out[:, :32]).any()
        ref, bound = attend(q[0], held[0][0], np.concatenate([np.zeros((n, 1, 32)), held[0][1][:, :, 32:]], -1))
        assert (np.abs(out - ref)[:, 32:] <= bound[:, 32:]).all()
    kv.free()


FIRST_CALLS = '''
import sys
import torch
import ssdllm
wtype, d = int(sys.argv[1]), int(sys.argv[2])
ctx = ssdllm.Context(0)
dev = torch.device("cuda", 0)
kv = ssdllm.PagedKvCache(ctx, 4, 16, 2, d, wtype)
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
table, pos, length, seq = i32([[0, 1, 2, 3]]), i32([5]), i32([6]), i32([0])
work = kv.attention_workspace()
bufs = []
for off in (0, 1):  # rows on 16-byte boundaries, and not
    for group in (4, 8):
        w = [torch.randn(1, n + 1, device=dev)[:, off:off + n] for n in (2 * d, 2 * d, 2 * group * d, 2 * group * d)]
        bufs.append(w + [torch.empty(1, 2 * d + 1, device=dev)[:, off:off + 2 * d] for _ in range(2)] +
                    [torch.full((1, 2 * group * d + 1), float("nan"), device=dev)[:, off:off + 2 * group * d]])
torch.cuda.synchronize()
def calls():
    for k, v, q, qo, ko, vo, out in bufs:
        kv.append(k, v, pos, table, seq=seq, q=q, q_out=qo)
        kv.read(pos, table, ko, vo, seq=seq)
        kv.attention(qo, length, table, out, work, seq=seq)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for b in bufs for t in b[3:]]
assert all(torch.isfinite(t).all() for t in got)
calls()
torch.cuda.synchronize()
assert all(torch.equal(a, t) for a, t in zip(got, [t for b in bufs for t in b[3:]]))
assert ctx.device_status() == 0
'''


@pytest.mark.parametrize("wtype,d", [(F16, 64), (BF16, 128), (Q8, 128), (Q4, 96)])
def test_the_first_calls_on_a_cache_may_be_captured(ctx, wtype, d):
    """In a process of its own: whatever the group of queries and the rows' alignment are, no call on
    the cache has to come before a capture."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ssd-llm_b200")
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS, str(wtype), str(d)], capture_output=True, text=True,
                       timeout=120, env={**os.environ, "PYTHONPATH": root, "CUDA_MODULE_LOADING": "LAZY"})
    assert r.returncode == 0, r.stderr[-2000:]


def test_the_largest_call_is_what_the_header_says(ctx):
    """n_rows (P / 16 + 4) n_head_kv ceil(group / 8) below 2^31: one row more is refused."""
    hk, group, pages = 2, 25, 1 << 22
    kv = ssdllm.PagedKvCache(ctx, 2, 16, hk, 64, Q8)
    table = torch.zeros(1, pages, dtype=torch.int32, device=DEV)
    work = kv.attention_workspace()
    for window in (0, 1 << 25):
        most = (2 ** 31 - 1) // (((window or pages * 16) // 16 + 4) * hk * 4)
        for n in (most, most + 1):
            q = torch.zeros(n, hk * group * 64, device=DEV)
            out, none = torch.full_like(q, float("nan")), i32([0] * n)
            if n > most:
                assert status(kv.attention, q, none, table, out, work, seq=none, window=window) == 3
            else:
                kv.attention(q, none, table, out, work, seq=none, window=window)
                assert (out == 0).all()
    kv.free()


@pytest.mark.parametrize("wtype", TYPES)
def test_a_chain_of_calls_under_programmatic_launch(ctx, wtype):
    """Append, attention and read one after the other, each on what the one before wrote, many times
    over: the bits of launches without it."""
    rng = np.random.default_rng(31)
    n, hk, h, d = 70, 2, 8, 64
    x = torch.from_numpy(rng.standard_normal((n, (h + 2 * hk) * d)).astype(np.float32)).to(DEV)
    table, work = i32([[4, 0, 2, 1, 3]]), None
    got = []
    try:
        for on in (False, True):
            ctx.set_pdl(on)
            kv = ssdllm.PagedKvCache(ctx, 5, 16, hk, d, wtype)
            work = kv.attention_workspace()
            q, out, o = torch.empty(1, h * d, device=DEV), torch.zeros(n, h * d, device=DEV), torch.zeros(2, n, hk * d, device=DEV)
            ints, seq = i32(np.arange(n + 1)), i32([0])
            torch.cuda.synchronize()
            for p in range(n):
                at = ints[p:p + 1]
                row = x[p:p + 1]
                kv.append(row[:, h * d:(h + hk) * d], row[:, (h + hk) * d:], at, table, seq=seq, q=row[:, :h * d], q_out=q)
                kv.attention(q, ints[p + 1:p + 2], table, out[p:p + 1], work, seq=seq)
                kv.read(at, table, o[0, p:p + 1], o[1, p:p + 1], seq=seq)
            torch.cuda.synchronize()
            got.append((out, o))
            kv.free()
    finally:
        ctx.set_pdl(False)
    assert torch.isfinite(got[0][0]).all() and (got[0][1] != 0).any(-1).all()
    for a, b in zip(*got):
        assert torch.equal(a, b)
