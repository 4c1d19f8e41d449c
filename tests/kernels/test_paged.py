"""Paged-cache operators on the GPU against 64-bit oracles: page plan, QK-norm + rotation + append, and
single-token attention over pages.

Tolerances. Outputs are rounded once to their type (to nearest: at most half of the type's eps times
|out|, 2^-8 for bf16 and 2^-11 for fp16). Attention: a score is a dot product of at most 256 exact products accumulated in fp32;
with |q|, |k| near sqrt(D) its error is below 256 * 2^-24 * D * scale <= 2^-12, so each probability is
off by a factor within 1 +- 2^-12 in the numerator and the denominator, 2^-11 * sum(p |v|) together
(probabilities split into two 16-bit terms and fp32 sums stay below that). Norm and rotation: a rotated
element is a sum of two products; fp32 rounding, the approximate reciprocal square root and the square
sum stay below 2^-20 of |a| + |b|."""

import math

import pytest
import torch

from mint_b200.ops import _ext, paged_attention, paged_plan, qk_norm_rope_paged

pytestmark = pytest.mark.gpu

U = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}


@pytest.fixture(autouse=True)
def _clean_status():
    _ext.reset_fallbacks()
    yield
    assert not _ext.fallback_counts()
    _ext.check_device_status()


def make_cache(lens, hkv, dim, page, dtype, layout="hnd", seed=0, extra=3, width_extra=1):
    """Pools full of NaN with the requests' keys written to shuffled pages -> k, v, tables, and the keys."""
    g = torch.Generator().manual_seed(seed)
    counts = [(n + page - 1) // page for n in lens]
    pool = sum(counts) + extra
    ids = torch.randperm(pool, generator=g).tolist()
    width = max(counts + [1]) + width_extra
    tables = torch.randint(-5, pool + 5, (len(lens), width), generator=g, dtype=torch.int32)  # unused entries: junk
    shape = (pool, hkv, page, dim) if layout != "nhd" else (pool, page, hkv, dim)
    if layout == "sliced":  # one layer of a two-layer pool that holds K and V side by side
        big = torch.full((pool, 2, 2, hkv, page, dim), float("nan"), dtype=dtype)
        kp, vp = big[:, 1, 0], big[:, 1, 1]
    else:
        kp = torch.full(shape, float("nan"), dtype=dtype)
        vp = torch.full(shape, float("nan"), dtype=dtype)
        if layout == "nhd":
            kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    keys = []
    at = 0
    for b, n in enumerate(lens):
        k = torch.randn(n, hkv, dim, generator=g).to(dtype)
        v = torch.randn(n, hkv, dim, generator=g).to(dtype)
        for c in range(counts[b]):
            pid = ids[at]
            at += 1
            tables[b, c] = pid
            m = min(page, n - c * page)
            kp[pid, :, :m] = k[c * page : c * page + m].transpose(0, 1)
            vp[pid, :, :m] = v[c * page : c * page + m].transpose(0, 1)
        keys.append((k, v))
    if layout == "sliced":
        big = big.cuda()
        return big[:, 1, 0], big[:, 1, 1], tables.cuda(), keys
    if layout == "nhd":
        return kp.transpose(1, 2).contiguous().cuda().transpose(1, 2), vp.transpose(1, 2).contiguous().cuda().transpose(1, 2), tables.cuda(), keys
    return kp.cuda(), vp.cuda(), tables.cuda(), keys


def oracle(q, keys, positions, rows, window, slopes, scale):
    """(output, sum p|v|) in 64 bits, one query and head at a time."""
    n, hq, d = q.shape
    out, mag = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64)
    for i in range(n):
        pos, row = int(positions[i]), int(rows[i])
        if pos < 0 or row < 0:
            continue
        k, v = keys[row]
        lo = max(0, pos - window) if window >= 0 else 0
        g = hq // k.shape[1]
        for h in range(hq):
            kk, vv = k[lo : pos + 1, h // g].double(), v[lo : pos + 1, h // g].double()
            s = kk @ q[i, h].double() * scale
            if slopes is not None:
                s = s + slopes[h].double() * (torch.arange(lo, pos + 1).double() - pos)
            p = torch.softmax(s, 0)
            out[i, h], mag[i, h] = p @ vv, p @ vv.abs()
    return out, mag


def check_attention(lens, hq, hkv, dim, page, *, window=-1, alibi=False, dtype=torch.bfloat16, layout="hnd", rows=None,
                    positions=None, scale=None, seed=0):
    kp, vp, tables, keys = make_cache(lens, hkv, dim, page, dtype, layout, seed)
    g = torch.Generator().manual_seed(seed + 1)
    rows_l = list(range(len(lens))) if rows is None else rows
    pos_l = [n - 1 for n in lens] if positions is None else positions
    q = torch.randn(len(rows_l), hq, dim, generator=g).to(dtype)
    slopes = torch.exp2(-8.0 * torch.arange(1, hq + 1) / hq) if alibi else None
    args = (q.cuda(), kp, vp, tables, torch.tensor(pos_l, dtype=torch.int32, device="cuda"),
            None if rows is None else torch.tensor(rows_l, dtype=torch.int32, device="cuda"))
    kw = {"window_left": window, "alibi_slopes": None if slopes is None else slopes.cuda(), "scale": scale}
    got = paged_attention(*args, **kw)
    again = paged_attention(*args, **kw)
    assert torch.equal(got, again)
    want, mag = oracle(q, keys, pos_l, rows_l, window, slopes, scale if scale is not None else 1 / math.sqrt(dim))
    err = (got.cpu().double() - want).abs()
    tol = U[dtype] * want.abs() + 2.0**-11 * mag + 1e-7
    assert bool((err <= tol).all()), f"worst excess {((err - tol).max()).item()}, err {err.max().item()}"


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 6), (16, 4), (12, 1), (9, 3)])
def test_attention_heads_types(dim, dtype, hq, hkv):
    check_attention([1, 2, 63, 64, 65, 200, 517], hq, hkv, dim, 16, dtype=dtype)


@pytest.mark.parametrize("hq,hkv", [(17, 1), (32, 1), (33, 1), (64, 1), (80, 1), (130, 1), (48, 2)])
def test_attention_wide_groups(hq, hkv):
    check_attention([1, 70, 333], hq, hkv, 128, 32)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("layout", ["hnd", "nhd", "sliced"])
def test_attention_pages_layouts(page, layout):
    check_attention([1, 7, 8, 9, 129, 1025, 2047], 4, 2, 128, page, layout=layout)


@pytest.mark.parametrize("window", [0, 1, 15, 16, 63, 64, 100, 511, 5000])
@pytest.mark.parametrize("page", [8, 64, 256])
def test_attention_window_ignores_older_keys(window, page):
    lens = [1, 2, 64, 65, 300, 1111]
    kp, vp, tables, keys = make_cache(lens, 2, 128, page, torch.bfloat16)
    for b, n in enumerate(lens):  # NaN wherever the window does not reach
        for j in range(max(0, n - 1 - window)):
            pid = int(tables[b, j // page])
            kp[pid, :, j % page] = float("nan")
            vp[pid, :, j % page] = float("inf")
    q = torch.randn(len(lens), 4, 128, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    pos = [n - 1 for n in lens]
    got = paged_attention(q.cuda(), kp, vp, tables, torch.tensor(pos, dtype=torch.int32, device="cuda"), window_left=window)
    want, mag = oracle(q, keys, pos, range(len(lens)), window, None, 1 / math.sqrt(128))
    err = (got.cpu().double() - want).abs()
    assert bool((err <= U[torch.bfloat16] * want.abs() + 2.0**-11 * mag + 1e-7).all())


@pytest.mark.parametrize("hq,hkv,dim", [(4, 4, 64), (12, 1, 64), (16, 4, 128), (6, 6, 256)])
@pytest.mark.parametrize("window", [-1, 100])
def test_attention_alibi(hq, hkv, dim, window):
    check_attention([1, 40, 700, 1500], hq, hkv, dim, 16, alibi=True, window=window, dtype=torch.float16)


def test_attention_packed_rows_padding_and_several_queries_per_request():
    lens = [300, 5, 77]
    rows = [2, 0, 0, 0, -1, 1, 2, 9, 0]
    positions = [76, 0, 150, 299, 12, -1, 3, 4, 298]
    kp, vp, tables, keys = make_cache(lens, 2, 128, 16, torch.bfloat16)
    q = torch.randn(len(rows), 8, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    i32 = {"dtype": torch.int32, "device": "cuda"}
    got = paged_attention(q.cuda(), kp, vp, tables, torch.tensor(positions, **i32), torch.tensor(rows, **i32))
    use = [r if r < 3 else -1 for r in rows]
    want, mag = oracle(q, keys, positions, use, -1, None, 1 / math.sqrt(128))
    err = (got.cpu().double() - want).abs()
    assert bool((err <= U[torch.bfloat16] * want.abs() + 2.0**-11 * mag).all())
    for i in (4, 5, 7):
        assert not got[i].any()


@pytest.mark.parametrize("n", [1, 2, 150, 700])
def test_attention_many_requests_and_long_tails(n):
    g = torch.Generator().manual_seed(n)
    lens = [int(x) for x in torch.randint(1, 90, (n,), generator=g)]
    lens[n // 2] = 9001  # one request far longer than the rest is split over the GPU
    check_attention(lens, 4, 2, 64, 16)


def test_attention_no_queries_and_idle_batch():
    kp, vp, tables, _ = make_cache([5, 6], 2, 128, 16, torch.bfloat16)
    q = torch.randn(0, 4, 128, device="cuda", dtype=torch.bfloat16)
    i32 = {"dtype": torch.int32, "device": "cuda"}
    empty = torch.empty(0, **i32)
    assert paged_attention(q, kp, vp, tables, empty, empty).shape == (0, 4, 128)
    q = torch.randn(2, 4, 128, device="cuda", dtype=torch.bfloat16)
    out = paged_attention(q, kp, vp, tables, torch.tensor([-1, -1], **i32))
    assert not out.any()


def test_attention_large_scores_do_not_overflow():
    kp, vp, tables, keys = make_cache([400], 1, 128, 16, torch.bfloat16)
    q = (300 * torch.randn(1, 2, 128, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16)
    got = paged_attention(q.cuda(), kp, vp, tables, torch.tensor([399], dtype=torch.int32, device="cuda"), scale=1.0)
    # scores of order 3e3 * sqrt(128): one key takes all the weight
    k, v = keys[0]
    s = k[:, 0].double() @ q[0].double().T
    best = s.argmax(0)
    assert bool((s.topk(2, dim=0).values.diff(dim=0).abs() > 30).all())
    assert torch.equal(got.cpu()[0], v[best, 0])


def test_attention_offsets_beyond_32_bits():
    page, hkv, dim = 64, 4, 128
    pool = 2**31 // (page * hkv * dim) + 8  # more than 2^31 elements
    kp = torch.empty(pool, hkv, page, dim, device="cuda", dtype=torch.bfloat16)
    vp = torch.empty_like(kp)
    ids = [pool - 1, 0, pool - 3]
    k, v = torch.randn(150, hkv, dim).to(torch.bfloat16), torch.randn(150, hkv, dim).to(torch.bfloat16)
    for c, pid in enumerate(ids):
        m = min(page, 150 - c * page)
        kp[pid, :, :m] = k[c * page : c * page + m].transpose(0, 1).cuda()
        vp[pid, :, :m] = v[c * page : c * page + m].transpose(0, 1).cuda()
    q = torch.randn(1, 8, dim).to(torch.bfloat16)
    i32 = {"dtype": torch.int32, "device": "cuda"}
    got = paged_attention(q.cuda(), kp, vp, torch.tensor([ids], **i32), torch.tensor([149], **i32))
    want, mag = oracle(q, [(k, v)], [149], [0], -1, None, 1 / math.sqrt(dim))
    err = (got.cpu().double() - want).abs()
    assert bool((err <= U[torch.bfloat16] * want.abs() + 2.0**-11 * mag).all())
    # the append writes its line of the last page
    qkv = torch.randn(1, (8 + 2 * hkv) * dim, device="cuda", dtype=torch.bfloat16)
    one = torch.zeros(dim, device="cuda")
    slot = torch.tensor([(pool - 1) * page + 63], **i32)
    qk_norm_rope_paged(qkv, 8, hkv, dim, one, one, None, None, torch.tensor([0], **i32), slot, kp, vp)
    assert torch.equal(vp[pool - 1, :, 63], qkv.view(-1, dim)[8 + hkv :])


@pytest.mark.parametrize("with_rows", [True, False])
def test_attention_very_wide_tables(with_rows):
    """Tables for 2^30 keys per request: the queries go in several launches so that tile numbers fit an int."""
    page, n = 1024, 40
    lens = [1 + 97 * i % 700 for i in range(4 if with_rows else n)]
    kp, vp, tables, keys = make_cache(lens, 8, 64, page, torch.bfloat16)
    wide = torch.zeros(len(lens), 2**20, dtype=torch.int32, device="cuda")
    wide[:, : tables.shape[1]] = tables
    rows = [i % 4 for i in range(n)] if with_rows else list(range(n))
    pos = [lens[r] - 1 - i % min(3, lens[r]) for i, r in enumerate(rows)]
    q = torch.randn(n, 16, 64, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    i32 = {"dtype": torch.int32, "device": "cuda"}
    got = paged_attention(q.cuda(), kp, vp, wide, torch.tensor(pos, **i32), torch.tensor(rows, **i32) if with_rows else None)
    want, mag = oracle(q, keys, pos, rows, -1, None, 1 / 8)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= U[torch.bfloat16] * want.abs() + 2.0**-11 * mag + 1e-7).all())


def test_one_page_pools_with_odd_strides_of_single_dimensions():
    i32 = {"dtype": torch.int32, "device": "cuda"}
    flat = torch.randn(2, 8, 64, device="cuda", dtype=torch.bfloat16)
    kp, vp = (flat[i].as_strided((1, 1, 8, 64), (3, 5, 64, 1)) for i in (0, 1))
    q = torch.randn(1, 1, 64, device="cuda", dtype=torch.bfloat16)
    one_column = torch.zeros(1, 3, **i32)[:, :1]
    got = paged_attention(q, kp, vp, one_column, torch.tensor([4], **i32))
    want, mag = oracle(q.cpu(), [(flat[0, :, None].cpu(), flat[1, :, None].cpu())], [4], [0], -1, None, 1 / 8)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= U[torch.bfloat16] * want.abs() + 2.0**-11 * mag + 1e-7).all())


def test_attention_on_a_side_stream():
    kp, vp, tables, keys = make_cache([2000] * 4, 2, 128, 16, torch.bfloat16)
    q = torch.randn(4, 4, 128, device="cuda", dtype=torch.bfloat16)
    pos = torch.full((4,), 1999, dtype=torch.int32, device="cuda")
    want = paged_attention(q, kp, vp, tables, pos)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [paged_attention(q, kp, vp, tables, pos) for _ in range(20)]
    s.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_attention_in_a_cuda_graph_follows_the_lengths():
    kp, vp, tables, keys = make_cache([1500, 1500], 2, 128, 16, torch.bfloat16)
    q = torch.randn(2, 4, 128, device="cuda", dtype=torch.bfloat16)
    pos = torch.tensor([3, 1499], dtype=torch.int32, device="cuda")
    paged_attention(q, kp, vp, tables, pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, kp, vp, tables, pos)
    for a, b in ((3, 1499), (1000, 0), (-1, 700)):
        pos.copy_(torch.tensor([a, b], dtype=torch.int32))
        graph.replay()
        want, mag = oracle(q.cpu(), keys, [a, b], [0, 1], -1, None, 1 / math.sqrt(128))
        err = (out.cpu().double() - want).abs()
        assert bool((err <= U[torch.bfloat16] * want.abs() + 2.0**-11 * mag).all())


# ---------------------------------------------------------------------------------- append
def append_oracle(x, n_q, n_kv, qs, ks, cos, sin, positions):
    """q, k, v in 64 bits and the magnitude |a| + |b| of each rotated element."""
    x = x.double()
    outs = []
    for part, scale in ((x[:, :n_q], qs), (x[:, n_q : n_q + n_kv], ks)):
        y = part / torch.sqrt(part.pow(2).mean(-1, keepdim=True) + 1e-6) * (1 + scale.double())
        mag = y.abs()
        if cos is not None:
            half = y.shape[-1] // 2
            c, s = cos.double()[positions.clamp(min=0)][:, None], sin.double()[positions.clamp(min=0)][:, None]
            a, b = y[..., :half], y[..., half:]
            mag = (a.abs() + b.abs()).repeat(1, 1, 2)
            y = torch.cat([a * c - b * s, a * s + b * c], -1)
        outs.append((y, mag))
    return outs[0], outs[1], x[:, n_q + n_kv :]


@pytest.mark.parametrize("n,n_q,n_kv,dim,page,rope,dtype", [
    (1, 6, 6, 128, 16, True, torch.bfloat16), (1, 1, 1, 64, 8, True, torch.float16),
    (7, 16, 4, 128, 16, True, torch.bfloat16), (33, 3, 1, 256, 64, True, torch.bfloat16),
    (257, 8, 2, 64, 32, True, torch.float16), (1001, 5, 5, 128, 128, False, torch.bfloat16),
    (4099, 12, 1, 64, 16, True, torch.bfloat16), (130, 4, 2, 256, 8, False, torch.float16),
])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_append(n, n_q, n_kv, dim, page, rope, dtype, layout):
    g = torch.Generator().manual_seed(n)
    span = 300
    wide = torch.randn(n, (n_q + 2 * n_kv) * dim + 8, generator=g).to(dtype)  # rows with a stride of their own
    x = wide[:, : (n_q + 2 * n_kv) * dim]
    qs, ks = 0.2 * torch.randn(dim, generator=g), 0.2 * torch.randn(dim, generator=g)
    ang = torch.rand(span, dim // 2, generator=g) * 6.28
    cos, sin = (ang.cos(), ang.sin()) if rope else (None, None)
    pool = (n + page - 1) // page + 2
    positions = torch.randint(0, span, (n,), generator=g)
    slots = torch.randperm(pool * page, generator=g)[:n]
    if n > 4:
        positions[1] = -1  # padding: zero output, nothing stored
        slots[1] = -1
        slots[3] = -1  # a token that is not kept
    shape = (pool, n_kv, page, dim) if layout == "hnd" else (pool, page, n_kv, dim)
    kp0, vp0 = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
    kp, vp = kp0.cuda(), vp0.cuda()
    kpv, vpv = (kp, vp) if layout == "hnd" else (kp.transpose(1, 2), vp.transpose(1, 2))
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    q, k, v = qk_norm_rope_paged(wide.cuda()[:, : x.shape[1]], n_q, n_kv, dim, dev(qs), dev(ks), dev(cos), dev(sin),
                                 positions.int().cuda(), slots.int().cuda(), kpv, vpv, return_kv=True)
    (wq, mq), (wk, mk), wv = append_oracle(x.reshape(n, -1, dim), n_q, n_kv, qs, ks, cos, sin, positions)
    dead = positions < 0
    for w in (wq, wk, wv, mq, mk):
        w[dead] = 0
    for got, want, mag in ((q, wq, mq), (k, wk, mk)):
        err = (got.cpu().double() - want).abs()
        assert bool((err <= U[dtype] * want.abs() + 2.0**-20 * mag + 1e-7).all()), err.max()
    assert torch.equal(v.cpu().double(), wv)
    want_k, want_v = kp0.clone(), vp0.clone()
    wkv, wvv = (want_k, want_v) if layout == "hnd" else (want_k.transpose(1, 2), want_v.transpose(1, 2))
    for i in range(n):
        s = int(slots[i])
        if s >= 0:
            wkv[s // page, :, s % page] = k[i].cpu()
            wvv[s // page, :, s % page] = v[i].cpu()
    assert torch.equal(kp.cpu(), want_k) and torch.equal(vp.cpu(), want_v)
    q2 = qk_norm_rope_paged(wide.cuda()[:, : x.shape[1]], n_q, n_kv, dim, dev(qs), dev(ks), dev(cos), dev(sin),
                            positions.int().cuda(), slots.int().cuda(), kpv, vpv)
    assert torch.equal(q, q2)


def test_append_reports_positions_and_slots_out_of_range():
    page, dim = 16, 128
    kp = torch.zeros(2, 1, page, dim, device="cuda", dtype=torch.bfloat16)
    vp = torch.zeros_like(kp)
    one = torch.zeros(dim, device="cuda")
    table = torch.ones(4, dim // 2, device="cuda")
    i32 = {"dtype": torch.int32, "device": "cuda"}
    x = torch.randn(3, 3 * dim, device="cuda", dtype=torch.bfloat16)
    for pos, slot in (([0, 4, 1], [0, 1, 2]), ([0, 1, 2], [0, 32, 1])):
        kp.zero_()
        q = qk_norm_rope_paged(x, 1, 1, dim, one, one, table, table, torch.tensor(pos, **i32), torch.tensor(slot, **i32), kp, vp)
        with pytest.raises(_ext.DeviceStatusError):
            _ext.check_device_status()
        assert bool(q[0].any()) and bool(kp[0, 0, 0].any())
        assert int(kp.view(2, -1, dim).abs().sum(-1).ne(0).sum()) == 2


# ------------------------------------------------------------------------------------- plan
def plan_oracle(seq, new, tables, free, head, page, n_tokens):
    tables = [list(r) for r in tables]
    pos, slots, rows, ends = [], [], [], []
    for b in range(len(seq)):
        for p in range(seq[b], seq[b] + new[b]):
            if p % page == 0:
                tables[b][p // page] = free[head]
                head += 1
            pos.append(p)
            slots.append(tables[b][p // page] * page + p % page)
            rows.append(b)
        ends.append(len(pos))
    pad = [-1] * (n_tokens - len(pos))
    return pos + pad, slots + pad, rows + pad, ends, [s + n for s, n in zip(seq, new)], [head], tables


def make_plan(n, seq_hi, new_hi, page, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    seq = torch.randint(0, seq_hi + 1, (n,), generator=g).tolist()
    new = torch.randint(0, new_hi + 1, (n,), generator=g).tolist()
    width = max([(s + a + page - 1) // page for s, a in zip(seq, new)] + [1]) + 1
    have = [(s + page - 1) // page for s in seq]
    need = sum((s + a + page - 1) // page for s, a in zip(seq, new)) - sum(have)
    ids = torch.randperm(sum(have) + need + 5, generator=g).tolist()
    tables = [[-7] * width for _ in range(n)]
    at = 0
    for b in range(n):
        tables[b][: have[b]] = ids[at : at + have[b]]
        at += have[b]
    return seq, new, tables, ids, at, sum(new) + pad


@pytest.mark.parametrize("n,seq_hi,new_hi,page,pad", [
    (1, 0, 1, 16, 0), (1, 40, 1, 8, 3), (5, 100, 1, 16, 5), (37, 64, 40, 16, 0), (300, 500, 1, 16, 300),
    (257, 0, 900, 32, 0), (1000, 33, 3, 8, 17), (2049, 100, 2, 64, 0), (16384, 20, 1, 16, 9), (3, 0, 70000, 1024, 0),
])
def test_plan(n, seq_hi, new_hi, page, pad):
    seq, new, tables, free, head, n_tokens = make_plan(n, seq_hi, new_hi, page, n, pad)
    if n == 1 and new_hi == 1:
        new, n_tokens = [1], 1 + pad
    i32 = {"dtype": torch.int32, "device": "cuda"}
    t = torch.tensor(tables, **i32)
    args = (torch.tensor(seq, **i32), torch.tensor(new, **i32), t, torch.tensor(free, **i32), torch.tensor([head], **i32))
    want = plan_oracle(seq, new, tables, free, head, page, n_tokens)
    for _ in range(2):  # the second call finds its own entries in the tables
        got = paged_plan(*args, page_size=page, n_tokens=n_tokens)
        for name, a, b in zip(got._fields, got, want):
            assert a.dtype == torch.int32 and a.tolist() == b, name
        assert t.tolist() == want[-1]


def test_plan_takes_strided_tables_and_leaves_the_rest_alone():
    i32 = {"dtype": torch.int32, "device": "cuda"}
    big = torch.full((6, 10), -9, **i32)
    got = paged_plan(torch.tensor([0, 16], **i32), torch.tensor([17, 1], **i32), big[1:5:2, 2:6],
                     torch.arange(20, **i32), torch.tensor([4], **i32), page_size=16, n_tokens=18)
    assert int(got.free_head) == 7
    want = torch.full((6, 10), -9, **i32)
    want[1, 2], want[1, 3], want[3, 3] = 4, 5, 6
    assert torch.equal(big, want)


@pytest.mark.parametrize("what", ["pages", "width", "tokens", "negative", "huge"])
def test_plan_reports_what_it_cannot_place(what):
    i32 = {"dtype": torch.int32, "device": "cuda"}
    seq, new, n_tokens, width, head = [0, 3], [20, 2], 22, 4, 0
    if what == "pages":
        head = 18
    elif what == "width":
        width = 1
    elif what == "tokens":
        n_tokens = 21
    elif what == "negative":
        new = [20, -2]
    else:
        seq = [2**31 - 1, 3]
    tables = torch.full((2, width), 19, **i32)
    got = paged_plan(torch.tensor(seq, **i32), torch.tensor(new, **i32), tables, torch.arange(20, **i32),
                     torch.tensor([head], **i32), page_size=8, n_tokens=n_tokens)
    torch.cuda.synchronize()
    with pytest.raises(_ext.DeviceStatusError):
        _ext.check_device_status()
    slots = got.slots.tolist()
    assert all(-1 <= s < 160 for s in slots)
    if what == "pages":  # two pages left: tokens 0..15 have slots, 16..19 have none
        assert slots[:16] == list(range(144, 160)) and slots[16:20] == [-1] * 4 and int(got.free_head) == 20
    if what == "width":
        assert slots[:8] == list(range(8)) and slots[8:20] == [-1] * 12


# -------------------------------------------------------------------------------- refusals
def test_refusals():
    kp, vp, tables, _ = make_cache([5, 6], 2, 128, 16, torch.bfloat16)
    q = torch.randn(2, 4, 128, device="cuda", dtype=torch.bfloat16)
    i32 = {"dtype": torch.int32, "device": "cuda"}
    pos = torch.tensor([4, 5], **i32)
    for bad in (
        lambda: paged_attention(q, kp, vp, tables, pos.long()),
        lambda: paged_attention(q, kp, vp, tables, pos.cpu()),
        lambda: paged_attention(q, kp, vp, tables.long(), pos),
        lambda: paged_attention(q, kp, vp[:3], tables, pos),
        lambda: paged_attention(q, kp, vp, tables, pos[:1]),
        lambda: paged_attention(q, kp, vp, tables, pos, pos[:1]),
        lambda: paged_attention(q, kp, vp, tables, pos, alibi_slopes=torch.ones(3, device="cuda")),
        lambda: paged_attention(q, kp.transpose(2, 3).contiguous().transpose(2, 3), vp, tables, pos),
        lambda: paged_plan(pos, pos, tables.cpu(), pos, pos[:1], page_size=16, n_tokens=2),
        lambda: paged_plan(pos, pos[:1], tables, pos, pos[:1], page_size=16, n_tokens=2),
        lambda: paged_plan(pos, pos, tables, pos, pos[:1], page_size=16, n_tokens=-1),
        lambda: paged_plan(pos.long(), pos, tables, pos, pos[:1], page_size=16, n_tokens=2),
    ):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
