"""The paged 4-bit KV cache on the GPU against its 64-bit restatement (oracle/kv4_oracle.py).

Writing and reading are exact: every value equals the restatement's.  Page management is exact.  Attention is compared with
64-bit softmax attention over the same dequantised values; its tolerance counts, with A = sum p |v| of the output element,
  bfloat16: half a step of the output (2^-8 |o|) and of every probability before its product with v (2^-8 A);
  both:     float32 sums of hd terms in a score, each product and sum off by at most 2^-23 of what has been summed
            (e = hd 2^-23 scale sum |q k|, twice: numerator and normaliser), and of the row's keys (T 2^-23 A);
  bfloat16: one kernel sums key codes with an offset and takes it off again.  A key's group enters as 128 + u with u <= 15 and
            -136 sum q: what is summed is at most 143 s |q| a channel, over 33 terms (2 * 33 * 2^-23 scale sum 143 s |q|
            for A).
"""
import random

import pytest
import torch

from oracle import kv4_oracle as K

pytestmark = pytest.mark.gpu
PAGE = 64


def _cache(layers, pages, rows, max_len, heads, hd, fill=None):
    from jaxml_b200 import PagedKVCache

    c = PagedKVCache.init(layers, pages, rows, max_len, heads, hd)
    if fill is not None:
        c.pages.fill_(fill)
    return c


class _Rows(list):
    """Dequantised rows, and their scales spread over the channels."""

    def __init__(self, xs):
        super().__init__(K.dequantised(x) for x in xs)
        self.scale = [K.quantise(x)[1].repeat_interleave(32, -1) for x in xs]


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


# -- writing and reading ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,heads,rows,S,before", [(64, 3, 2, 1, 0), (128, 8, 5, 1, 63), (256, 1, 3, 5, 61),
                                                    (128, 2, 4, 130, 1), (64, 8, 1, 64, 64), (256, 4, 2, 67, 0)])
def test_append_and_read_are_exact(dtype, hd, heads, rows, S, before):
    c = _cache(2, rows * 8 + 3, rows, 8 * PAGE, heads, hd, fill=0xA5)
    history = [torch.zeros(0, heads, hd, dtype=torch.float64) for _ in range(rows)], [
        torch.zeros(0, heads, hd, dtype=torch.float64) for _ in range(rows)]
    for call, (n, seed) in enumerate(((before, 1), (S, 2))):
        if n == 0:
            continue
        counts = [n if r % 3 == 0 else max(0, n - r) for r in range(rows)]
        k, v = _rand((rows, n, heads, hd), dtype, seed, 3.0), _rand((rows, n, heads, hd), dtype, seed + 10, 0.01)
        for r in range(rows):      # what stands behind a row's tokens is not read
            k[r, counts[r]:], v[r, counts[r]:] = float("nan"), float("inf")
        c.extend(torch.tensor(counts, dtype=torch.int32, device="cuda"))
        c.append(1, k.cuda(), v.cuda())
        for x, h in ((k, history[0]), (v, history[1])):
            for r in range(rows):
                h[r] = torch.cat([h[r], K.dequantised(x[r, :counts[r]])])
    c.check()
    lens = [h.shape[0] for h in history[0]]
    assert c.lengths.tolist() == lens
    for out_dtype in (torch.bfloat16, torch.float32):
        got = c.read(1, 0, max(lens) + 2, dtype=out_dtype)
        for x, h in zip(got, history):
            assert x.dtype == out_dtype
            for r in range(rows):
                assert torch.equal(x[r, :lens[r]].double().cpu(), h[r]), (r, out_dtype)
                assert (x[r, lens[r]:] == 0).all()
    start = c.lengths - c.counts
    tail = c.read(1, start, S, dtype=torch.float32)[0]
    for r in range(rows):
        n = min(S, lens[r] - int(start[r]))
        assert torch.equal(tail[r, :n].double().cpu(), history[0][r][int(start[r]):])
    assert (c.pages[0] == 0xA5).all()          # the other layer


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_takes_any_strides(dtype):
    """Heads out of a fused projection, a transposed sequence axis, a base off its 16-byte boundary, a broadcast row."""
    rows, S, heads, hd = 3, 5, 2, 64
    fused = _rand((rows, S, 3, heads, hd), dtype, 1).cuda()
    odd = _rand((rows * S * heads * hd + 1,), dtype, 2).cuda()[1:].view(rows, S, heads, hd)
    turned = _rand((S, rows, heads, hd), dtype, 3).cuda().transpose(0, 1)
    one = _rand((1, S, heads, hd), dtype, 4).cuda().expand(rows, S, heads, hd)
    spread = _rand((rows, S, heads, 2 * hd), dtype, 5).cuda()[..., ::2]
    wide = _rand((rows, S, heads, hd + 3), dtype, 6).cuda()[..., 2:2 + hd]
    for k, v in ((fused[:, :, 1], fused[:, :, 2]), (odd, turned), (one, spread), (wide, odd)):
        c = _cache(1, 6, rows, PAGE, heads, hd)
        c.extend(S)
        c.append(0, k, v)
        gk, gv = c.read(0, 0, S, dtype=torch.float32)
        assert torch.equal(gk.double().cpu(), K.dequantised(k.cpu())) and torch.equal(gv.double().cpu(), K.dequantised(v.cpu()))
        c.check()


def test_append_special_values():
    """Zero groups, half steps, subnormal and huge groups, NaN and infinities: each group is as the format says."""
    hd = 64
    x = torch.zeros(1, 12, 1, hd)
    x[0, 1, 0, :8] = torch.tensor([7.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 3.5])       # scale 1: ties to even
    x[0, 2, 0, :4] = torch.tensor([7 * 1.0625, 7.0, -7 * 1.0625, 0.53125])           # a scale half way between two
    x[0, 3, 0, 5] = float("nan")
    x[0, 4, 0, 40], x[0, 4, 0, 41] = float("inf"), float("-inf")
    x[0, 5, 0, :] = 2.0 ** 122
    x[0, 6, 0, :] = -(2.0 ** 122) * (1 - 2.0 ** -24)
    x[0, 7, 0, :32] = torch.arange(32) * 2.0 ** -126
    x[0, 8, 0, :32] = torch.arange(32) * 2.0 ** -149
    x[0, 9, 0, 0] = -0.0
    x[0, 10, 0, :32] = 7 * 1.875 * 2.0 ** -100 * torch.linspace(-1, 1, 32)
    x[0, 11, 0, 32:] = torch.linspace(-3, 8, 32)
    c = _cache(1, 2, 1, PAGE, 1, hd)
    c.extend(12)
    c.append(0, x.cuda(), x.cuda())
    want = K.dequantised(x)
    for dtype in (torch.float32, torch.bfloat16):
        for got in c.read(0, 0, 12, dtype=dtype):
            g = got.double().cpu()
            assert torch.equal(torch.isnan(g), torch.isnan(want))
            assert torch.equal(g.nan_to_num(0), want.nan_to_num(0))
    assert torch.isnan(want[0, [3, 4, 5]]).sum() == 32 + 32 + 64 and not torch.isnan(want[0, 6:]).any()


# -- attention ----------------------------------------------------------------------------------------------------
def _filled(rows, lens, counts, heads, hd, seed, fill=0xFF, extra=3, peaky=1.0, room=0):
    """A cache whose rows hold lens tokens, the last counts of them the current call's; unused pages and slots hold NaN
    scales; tables have room for that many pages more than the rows need (long tables take another kernel).  Returns it
    and the rows' dequantised keys and values."""
    width = max(1, -(-max(lens) // PAGE)) + room
    c = _cache(1, sum(-(-n // PAGE) for n in lens) + extra, rows, width * PAGE, heads, hd, fill=fill)
    dev = torch.device("cuda")
    older = [n - k for n, k in zip(lens, counts)]
    k_all, v_all = _rand((rows, max(lens), heads, hd), torch.float32, seed, peaky), _rand((rows, max(lens), heads, hd),
                                                                                          torch.float32, seed + 1)
    for first, n in ((torch.zeros(rows, dtype=torch.int64), older), (torch.tensor(older), counts)):
        m = max(n)
        if m == 0 and first.sum() == 0:
            continue
        c.extend(torch.tensor(n, dtype=torch.int32, device=dev))
        if m == 0:
            continue
        at = (first[:, None] + torch.arange(m)[None]).clamp(max=max(lens) - 1)
        pick = lambda x: torch.gather(x, 1, at[:, :, None, None].expand(rows, m, heads, hd)).cuda()  # noqa: E731
        c.append(0, pick(k_all), pick(v_all))
    c.check()
    assert c.lengths.tolist() == list(lens) and c.counts.tolist() == list(counts)
    return c, _Rows([k_all[r, :lens[r]] for r in range(rows)]), _Rows([v_all[r, :lens[r]] for r in range(rows)])


def _check_attend(got, q, ks, vs, lens, counts, scale, window=0):
    hd = q.shape[-1]
    G = q.shape[2] // ks[0].shape[1]
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    for r in range(q.shape[0]):
        want = K.attend(q[r].double(), ks[r], vs[r], lens[r], counts[r], scale, window)
        A = K.attend(q[r].double(), ks[r], vs[r].abs(), lens[r], counts[r], scale, window)
        n = counts[r]
        assert (got[r, n:] == 0).all()
        if n == 0:
            continue
        big = torch.einsum("shd,thd->sht", q[r, :n].double().abs(), ks[r].abs().repeat_interleave(G, 1)).amax(-1)
        e = 2 * hd * 2.0 ** -23 * abs(scale) * big[..., None] + lens[r] * 2.0 ** -23
        tol = A[:n] * e + 1e-30
        if q.dtype == torch.bfloat16:
            spread = torch.einsum("shd,thd->sht", q[r, :n].double().abs(), ks.scale[r].repeat_interleave(G, 1)).amax(-1)
            tol = tol + 2.0 ** -8 * (want[:n].abs() + A[:n]) + A[:n] * 2 * 33 * 2.0 ** -23 * abs(scale) * 143 * spread[..., None]
        err = (got[r, :n] - want[:n]).abs()
        assert (err <= tol).all(), (r, (err / tol).max())


SHAPES = [  # heads, kv heads, hd
    (8, 2, 128), (4, 4, 64), (16, 8, 256), (32, 8, 128), (3, 3, 64), (9, 1, 128), (14, 2, 64), (33, 1, 128), (5, 1, 256),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("lens,room", [([1], 0), ([64, 1, 63, 65], 0), ([0, 129, 700], 0), ([130] * 9, 0), ([1], 500),
                                       ([0, 129, 700, 1], 500)])
def test_single_token_attention(dtype, heads, kv, hd, lens, room):
    counts = [min(1, n) for n in lens]
    c, ks, vs = _filled(len(lens), lens, counts, kv, hd, seed=heads, room=room)
    q = _rand((len(lens), 1, heads, hd), dtype, 5, 1.5)
    got = c.attend(0, q.cuda())
    assert got.dtype == dtype and got.shape == q.shape
    _check_attend(got, q, ks, vs, lens, counts, hd ** -0.5)
    c.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 4, 64), (16, 8, 256), (6, 1, 64)])
@pytest.mark.parametrize("S,lens,counts", [(2, [2, 66], [2, 1]), (7, [7, 64, 200, 5], [7, 0, 6, 3]), (64, [64, 128], [64, 64]),
                                           (33, [300, 33], [33, 17]), (150, [150, 410], [149, 150])])
@pytest.mark.parametrize("room", [0, 500])
def test_chunks(dtype, heads, kv, hd, S, lens, counts, room):
    c, ks, vs = _filled(len(lens), lens, counts, kv, hd, seed=S, room=room)
    q = _rand((len(lens), S, heads, hd), dtype, 5)
    for r, n in enumerate(counts):
        q[r, n:] = float("nan")                # padding is not read into anything
    got = c.attend(0, q.cuda())
    _check_attend(got, q, ks, vs, lens, counts, hd ** -0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 300, 5000])
def test_sliding_window(dtype, window):
    for S, lens, counts in ((1, [1, 500, 64], [1, 1, 1]), (70, [70, 333, 100], [70, 69, 0])):
        for room in (0, 500):
            c, ks, vs = _filled(3, lens, counts, 2, 64, seed=window, room=room)
            q = _rand((3, S, 6, 64), dtype, 5)
            got = c.attend(0, q.cuda(), sliding_window=window)
            _check_attend(got, q, ks, vs, lens, counts, 64 ** -0.5, window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0])
def test_scales(dtype, scale):
    """No preference, a negative one, and scores so large that one key takes all."""
    lens, counts = [200, 65, 1], [1, 1, 1]
    c, ks, vs = _filled(3, lens, counts, 2, 128, seed=3)
    q = _rand((3, 1, 8, 128), torch.float32, 5).to(dtype)
    got = c.attend(0, q.cuda(), scale=scale)
    _check_attend(got, q, ks, vs, lens, counts, scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_query_strides(dtype):
    lens, counts = [100, 70], [3, 2]
    c, ks, vs = _filled(2, lens, counts, 2, 64, seed=4)
    fused = _rand((2, 3, 12, 64), dtype, 1).cuda()
    odd = _rand((2 * 3 * 8 * 64 + 1,), dtype, 2).cuda()[1:].view(2, 3, 8, 64)
    turned = _rand((8, 3, 2, 64), dtype, 3).cuda().transpose(0, 2)
    spread = _rand((2, 3, 8, 128), dtype, 4).cuda()[..., 1::2]
    one = _rand((1, 1, 8, 64), dtype, 5).cuda().expand(2, 3, 8, 64)
    for q in (fused[:, :, :8], fused[:, :, 1:9], odd, turned, spread, one):
        _check_attend(c.attend(0, q), q.cpu(), ks, vs, lens, counts, 64 ** -0.5)


def test_long_row_is_split_and_joined():
    """One row far longer than the others, and enough keys that many parts of it are summed."""
    lens, counts = [9001, 3], [1, 1]
    c, ks, vs = _filled(2, lens, counts, 1, 128, seed=8)
    for dtype in (torch.bfloat16, torch.float32):
        q = _rand((2, 1, 4, 128), dtype, 5)
        _check_attend(c.attend(0, q.cuda()), q, ks, vs, lens, counts, 128 ** -0.5)


@pytest.mark.parametrize("room", [0, 500])
def test_many_rows(room):
    """More rows than multiprocessors, most of them of one or two pages, some empty."""
    rng = random.Random(1)
    lens = [rng.choice([0, 1, 60, 64, 100, 140]) for _ in range(300)]
    counts = [min(1, n) if i % 7 else 0 for i, n in enumerate(lens)]
    c, ks, vs = _filled(300, lens, counts, 2, 64, seed=8, room=room)
    q = _rand((300, 1, 4, 64), torch.bfloat16, 5)
    _check_attend(c.attend(0, q.cuda()), q, ks, vs, lens, counts, 64 ** -0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("max_len,group", [(128, 1), (40000, 1), (128, 2), (40000, 4), (40000, 8)])
def test_a_visible_nan_is_seen_and_a_hidden_one_is_not(dtype, max_len, group):
    """A key or value group that decodes to NaN reaches the queries that see it, and no other row or query."""
    hd, heads = 64, 2
    c = _cache(1, 8, 2, max_len, heads, hd, fill=0xFF)
    k, v = _rand((2, 70, heads, hd), torch.float32, 1), _rand((2, 70, heads, hd), torch.float32, 2)
    k[0, 50, 1, 3] = float("nan")
    v[1, 69, 0, 40] = float("inf")
    c.extend(70)
    c.append(0, k.cuda(), v.cuda())
    q = _rand((2, 70, heads * group, hd), dtype, 3)
    got = torch.isnan(c.attend(0, q.cuda())).cpu()
    want = torch.zeros_like(got)
    want[0, 50:, group:] = True                 # its score is NaN: the whole softmax is
    want[1, 69, :group, 32:] = True             # its value is NaN in one group of channels
    assert torch.equal(got, want)
    got = torch.isnan(c.attend(0, q.cuda(), sliding_window=5)).cpu()
    want[0, 55:] = False
    assert torch.equal(got, want)
    got = torch.isnan(c.attend(0, q[:, -1:].cuda())).cpu()        # one query at a time: counts[r] tokens, the first here
    assert int(c.status.item()) == 4            # fewer queries than tokens is reported, and nothing is out of range
    c.status.zero_()
    c.rollback(1)
    c.extend(1)
    c.append(0, k[:, 69:].cuda(), v[:, 69:].cuda())
    got = torch.isnan(c.attend(0, q[:, -1:].cuda())).cpu()
    want = torch.zeros_like(got)
    want[0, 0, group:], want[1, 0, :group, 32:] = True, True
    assert torch.equal(got, want)


@pytest.mark.parametrize("room", [0, 500])
def test_page_ids_out_of_range_are_skipped_and_reported(room):
    c, ks, vs = _filled(2, [130, 130], [1, 1], 2, 64, seed=4, room=room)
    c.table[0, 1], c.table[0, 0] = 1 << 20, -7
    q = _rand((2, 1, 4, 64), torch.bfloat16, 5)
    got = c.attend(0, q.cuda())
    for x in (ks, vs):
        x[0], x.scale[0] = x[0][128:], x.scale[0][128:]
    _check_attend(got, q, ks, vs, [2, 130], [1, 1], 0.125)
    with pytest.raises(RuntimeError, match="device status 4"):
        c.check()
    c.check()
    c.append(0, _rand((2, 1, 2, 64), torch.bfloat16, 1).cuda(), _rand((2, 1, 2, 64), torch.bfloat16, 1).cuda())
    c.check()                                   # position 129 is on the third page
    c.table[0, 2] = c.num_pages
    c.append(0, _rand((2, 1, 2, 64), torch.bfloat16, 1).cuda(), _rand((2, 1, 2, 64), torch.bfloat16, 1).cuda())
    with pytest.raises(RuntimeError, match="device status 4"):
        c.check()
    assert (c.read(0, 129, 1)[0][0] == 0).all()
    with pytest.raises(RuntimeError, match="device status 4"):
        c.check()


def test_more_tokens_than_queries_is_reported():
    c, ks, vs = _filled(1, [70], [3], 2, 64, seed=4)
    c.attend(0, _rand((1, 2, 4, 64), torch.bfloat16, 5).cuda())
    with pytest.raises(RuntimeError, match="out of range"):
        c.check()


@pytest.mark.parametrize("lens", [[3000, 40, 700], [500, 40, 700]])
def test_results_do_not_change_from_run_to_run(lens):
    c, _, _ = _filled(3, lens, [1, 1, 1], 4, 128, seed=4)
    q = _rand((3, 1, 16, 128), torch.bfloat16, 5).cuda()
    want = c.attend(0, q)
    for _ in range(20):
        assert torch.equal(c.attend(0, q), want)


# -- pages --------------------------------------------------------------------------------------------------------
def _tables(c):
    return [[p for p in row if p >= 0] for row in c.table.tolist()]


@pytest.mark.parametrize("seed,rows,row_pages,pages", [(0, 5, 4, 16), (1, 1, 6, 9), (2, 40, 3, 90), (3, 3, 5, 700)])
def test_page_calls_match_the_restatement(seed, rows, row_pages, pages):
    """Random calls: tables, lengths, holders, the status and what the rows hold in two layers."""
    rng = random.Random(seed)
    hd, heads = 64, 1
    c, want = _cache(2, pages, rows, row_pages * PAGE, heads, hd), K.Pages(rows, row_pages, pages)
    g = torch.Generator().manual_seed(seed)
    tag = 0
    for _ in range(60):
        what = rng.choice(["extend", "extend", "extend", "fork", "rollback", "free", "compact"])
        if what == "extend":
            counts = [rng.choice([0, 1, 1, 3, 64, 70]) for _ in range(rows)]
            if rng.random() < 0.3:
                counts = [1] * rows
                c.extend(1)
            else:
                c.extend(torch.tensor(counts, dtype=rng.choice([torch.int32, torch.int64])))
            want.extend(counts)
            S = max(max(counts), 1)
            base = torch.randint(1, 8, (rows, S, heads, hd), generator=g).float() * 2.0 ** (tag % 20 - 10)
            base[..., 0], base[..., 32] = 7 * 2.0 ** (tag % 20 - 10), 7 * 2.0 ** (tag % 20 - 10)   # scale = the power of two
            c.append(0, base.cuda(), -base.cuda())
            c.append(1, -base.cuda(), base.cuda())
            for r in range(rows):
                for i in range(want.counts[r]):
                    want.write(r, want.lengths[r] - want.counts[r] + i, base[r, i])
            tag += 1
        elif what == "fork":
            parents = [rng.randrange(-1, rows) for _ in range(rows)]
            if rng.random() < 0.1:
                parents[rng.randrange(rows)] = rows + 5
            c.fork(torch.tensor(parents))
            want.fork(parents)
        elif what == "rollback":
            cut = [rng.randrange(0, n + 1) if rng.random() < 0.5 else 0 for n in want.lengths]
            if rng.random() < 0.1:
                cut[rng.randrange(rows)] = 10 ** 6
            if rng.random() < 0.3:
                cut = [1] * rows
                c.rollback(1)
            else:
                c.rollback(torch.tensor(cut))
            want.rollback(cut)
        elif what == "free":
            gone = [r for r in range(rows) if rng.random() < 0.3]
            if rng.random() < 0.5:
                c.free(gone)
            else:
                c.free(torch.tensor([r in gone for r in range(rows)]).cuda())
            want.free(gone)
        else:
            assert int(c.compact()) == want.compact()
        assert _tables(c) == want.table and c.lengths.tolist() == want.lengths, what
        assert c.refs.tolist() == want.refs(), what
        code = int(c.status.item())
        assert (code == 4) == want.error and code in (0, 4), what
        c.status.zero_()
        want.error = False
    for r in range(rows):
        n = want.lengths[r]
        if n == 0:
            continue
        held = torch.stack(want.row(r))
        for layer, sign in ((0, 1.0), (1, -1.0)):
            k, v = c.read(layer, 0, n, dtype=torch.float32)
            assert torch.equal(k[r].cpu(), sign * held) and torch.equal(v[r].cpu(), -sign * held)


def test_a_full_pool_changes_nothing_and_is_reported():
    c = _cache(1, 3, 2, 4 * PAGE, 1, 64)
    c.extend(65)                                # four pages of three
    with pytest.raises(RuntimeError, match="no room"):
        c.check()
    assert c.lengths.tolist() == [0, 0] and c.counts.tolist() == [0, 0] and c.refs.tolist() == [0, 0, 0]
    kv = _rand((2, 65, 1, 64), torch.bfloat16, 1).cuda()
    c.append(0, kv, kv)                         # nothing is there to be written
    assert (c.pages == 0).all() and (c.attend(0, kv) == 0).all()
    c.extend([65, 1])
    c.check()
    assert c.lengths.tolist() == [65, 1] and c.refs.tolist() == [1, 1, 1]
    c.extend([200, 0])                          # past the row's table
    with pytest.raises(RuntimeError, match="no room"):
        c.check()
    assert c.lengths.tolist() == [65, 1]
    c.extend([-1, 0])
    with pytest.raises(RuntimeError, match="no room"):
        c.check()
    big = c.resize(9)
    big.extend([100, 100])
    big.check()
    assert big.lengths.tolist() == [165, 101] and c.lengths.tolist() == [65, 1]


def test_forked_rows_part_when_they_are_written():
    c = _cache(1, 10, 3, 2 * PAGE, 1, 64)
    one = torch.full((3, 70, 1, 64), 7.0)
    c.extend([70, 0, 0])
    c.append(0, one.cuda(), one.cuda())
    c.fork([0, 0, 0])
    assert c.refs.tolist()[:2] == [3, 3] and _tables(c) == [[0, 1]] * 3
    c.extend([0, 1, 1])                         # rows 1 and 2 write, row 0 keeps the shared page
    new = torch.tensor([1.0, 2.0, 3.0]).view(3, 1, 1, 1).expand(3, 1, 1, 64) * 7
    c.append(0, new.cuda(), new.cuda())
    c.check()
    assert _tables(c) == [[0, 1], [0, 2], [0, 3]] and c.refs.tolist()[:4] == [3, 1, 1, 1]
    k = c.read(0, 0, 71, dtype=torch.float32)[0].cpu()[:, :, 0, 0]
    assert (k[:, :70] == 7).all() and k[:, 70].tolist() == [0, 14, 21]


# -- streams, graphs, the model -------------------------------------------------------------------------------------
def test_two_streams_read_one_cache():
    c, ks, vs = _filled(2, [4000, 70], [1, 1], 4, 128, seed=4)
    q = [_rand((2, 1, 16, 128), torch.bfloat16, s).cuda() for s in (5, 6)]
    want = [c.attend(0, x) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.attend(0, q[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in (0, 1) for x in got[i])


def _step(c, kv, q):
    c.extend(1)
    outs = []
    for layer in range(c.num_layers):
        c.append(layer, kv[layer], kv[layer])
        outs.append(c.attend(layer, q[layer]))
    return torch.stack(outs)


def test_a_captured_loop_gives_the_eager_results():
    """extend, append, attend, fork and rollback in graphs: replays go on from the device's state.  Two graphs share the cache."""
    def state():
        c = _cache(2, 24, 3, 256, 2, 64, fill=0xFF)
        c.extend([60, 3, 100])
        x = _rand((3, 100, 2, 64), torch.bfloat16, 1).cuda()
        for layer in range(2):
            c.append(layer, x, x)
        return c

    kv, q = torch.zeros(2, 3, 1, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 3, 1, 4, 64, dtype=torch.bfloat16,
                                                                                         device="cuda")
    parents = torch.tensor([0, 2, 2], dtype=torch.int32, device="cuda")
    a, b = state(), state()
    _step(b, kv, q)                             # loads what is loaded once
    b.fork(parents)
    b.rollback(1)
    b = state()
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out1 = _step(b, kv, q)
    with torch.cuda.graph(g2):
        b.fork(parents)
        out2 = _step(b, kv, q)
        b.rollback(1)
    for i in range(12):
        kv.copy_(_rand((2, 3, 1, 2, 64), torch.bfloat16, 10 + i))
        q.copy_(_rand((2, 3, 1, 4, 64), torch.bfloat16, 40 + i))
        if i % 3 == 2:
            a.fork(parents)
            want = _step(a, kv, q)
            a.rollback(1)
            g2.replay()
            got = out2
        else:
            want = _step(a, kv, q)
            g1.replay()
            got = out1
        assert torch.equal(got, want), i
        for x, y in ((a.table, b.table), (a.lengths, b.lengths), (a.refs, b.refs)):
            assert torch.equal(x, y), i
    a.check()
    b.check()


def _tiny(family):
    from jaxml_b200 import GemmaModelWithHead, GPTNeoXModelWithHead, LlamaModelWithHead, ModelConfig

    kw = dict(head_dim=64, hidden_size=256, num_heads=4, num_kv_heads=2, num_layers=2, max_position_embeddings=256,
              vocab_size=512, intermediate_ratio=(3, 1), norm_eps=1e-5, rope_theta=10000.0)
    if family == "gemma3":
        kw.update(sliding_window=20, sliding_window_pattern=2)
    if family == "neox":
        kw.update(num_kv_heads=4)
    cls = {"llama": LlamaModelWithHead, "neox": GPTNeoXModelWithHead, "gemma3": GemmaModelWithHead}[family]
    model = cls(ModelConfig(**kw), dtype=torch.float32)
    return model, model.init(0, std=0.08)


@pytest.mark.parametrize("family", ["llama", "neox", "gemma3"])
def test_a_model_runs_over_the_paged_cache(family):
    """A prompt at once, in chunks and token by token give the same logits (float32: 1e-4 relative, as between the
    framework's own paths), and a forked row goes on like its parent."""
    from jaxml_b200 import PagedKVCache

    model, params = _tiny(family)
    cfg = model.config
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, cfg.vocab_size, (2, 40), generator=g, dtype=torch.int32)
    new = lambda: PagedKVCache.init(cfg.num_layers, 12, 2, 128, cfg.num_key_value_heads, 64)  # noqa: E731
    whole = new()
    out = model.apply(params, ids, kv_caches=whole, use_cache=True)
    assert out.kv_caches is whole and out.logits.shape == (2, 40, cfg.vocab_size)
    chunks = new()
    parts = [model.apply(params, ids[:, a:b], kv_caches=chunks).logits for a, b in ((0, 17), (17, 18), (18, 40))]
    tol = 1e-4 * out.logits.abs().max()
    assert (torch.cat(parts, 1) - out.logits).abs().max() <= tol
    ragged = new()
    mask = torch.ones(2, 40, dtype=torch.bool)
    mask[1, 25:] = False
    got = model.apply(params, ids, attention_mask=mask, kv_caches=ragged).logits
    assert (got[0] - out.logits[0]).abs().max() <= tol and (got[1, :25] - out.logits[1, :25]).abs().max() <= tol
    assert ragged.lengths.tolist() == [40, 25]
    whole.fork([0, 0])
    step = model.apply(params, ids[:1, :1].expand(2, 1), kv_caches=whole).logits
    assert torch.equal(step[0], step[1])
    with pytest.raises(ValueError, match="must match the model"):
        model.apply(params, ids[:1], kv_caches=whole)
    with pytest.raises(NotImplementedError, match="position_ids"):
        model.apply(params, ids, position_ids=torch.arange(40)[None], kv_caches=whole)
    with pytest.raises(ValueError, match="max_position_embeddings"):
        model.apply(params, torch.zeros(2, 250, dtype=torch.int32), kv_caches=whole)
    full = PagedKVCache.init(cfg.num_layers, 1, 2, 128, cfg.num_key_value_heads, 64)
    with pytest.raises(RuntimeError, match="no room"):
        model.apply(params, ids, kv_caches=full)
    assert full.lengths.tolist() == [0, 0]


def test_beam_steps_with_scores():
    """The operators as a beam search uses them: prompt, then steps of score, choose, fork and go on."""
    from jaxml_b200 import PagedKVCache
    from jaxml_b200.sampling import token_log_probs

    model, params = _tiny("llama")
    cfg, beams, steps = model.config, 3, 4
    prompt = torch.randint(0, cfg.vocab_size, (1, 70), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    c = PagedKVCache.init(cfg.num_layers, 12, beams, 128, cfg.num_key_value_heads, 64)
    logits = model.apply(params, prompt.expand(beams, -1), kv_caches=c, keep_last_n_logits=1).logits[:, -1]
    c.fork([0] * beams)
    total, seqs = torch.tensor([0.0] + [float("-inf")] * (beams - 1), device="cuda"), [[] for _ in range(beams)]
    for _ in range(steps):
        s = token_log_probs(logits, torch.zeros(beams, dtype=torch.int32), top_n=beams)
        total, pick = (total[:, None] + s.top_log_probs).reshape(-1).topk(beams)
        parents, tok = pick // beams, s.top_ids.reshape(-1)[pick]
        c.fork(parents.to(torch.int32))
        seqs = [seqs[p] + [t] for p, t in zip(parents.tolist(), tok.tolist())]
        logits = model.apply(params, tok[:, None], kv_caches=c).logits[:, -1]
    c.check()
    assert c.lengths.tolist() == [70 + steps] * beams and len(set(map(tuple, seqs))) == beams
    # each beam's total is what scoring its tokens alone gives
    again = PagedKVCache.init(cfg.num_layers, 12, beams, 128, cfg.num_key_value_heads, 64)
    ids = torch.cat([prompt.expand(beams, -1), torch.tensor(seqs, dtype=torch.int32)], 1)
    lg = model.apply(params, ids, kv_caches=again).logits[:, 69:-1]
    lp = token_log_probs(lg, ids[:, 70:]).log_probs.sum(1)
    assert (lp - total).abs().max() <= 1e-3
    c.free([1])
    used = int(c.compact())
    assert used == len({p for t in _tables(c) for p in t})


# -- sizes at which another kernel or another split takes over ----------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,heads,lens", [(64, 2, [9 * PAGE, 0, 1, 200]), (128, 1, [17 * PAGE - 1, 30, 65, 700]),
                                           (256, 1, [33 * PAGE, 1, 500, 64]), (128, 3, [70 * PAGE + 1, 2, 64 * 3])])
@pytest.mark.parametrize("window", [0, 100])
def test_clusters_of_a_few_rows(dtype, hd, heads, lens, window):
    """A row's pages shared among 2, 4 and 8 CTAs: rows with fewer pages than CTAs, empty rows, a window that leaves most
    of the table unseen."""
    counts = [min(1, n) for n in lens]
    c, ks, vs = _filled(len(lens), lens, counts, heads, hd, seed=hd)
    q = _rand((len(lens), 1, heads * 4, hd), dtype, 5, 1.5)
    got = c.attend(0, q.cuda(), sliding_window=window or None)
    _check_attend(got, q, ks, vs, lens, counts, hd ** -0.5, window)
    assert torch.equal(got, c.attend(0, q.cuda(), sliding_window=window or None))
    c.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("S", [2, 4, 5, 16, 17, 32, 33])
def test_query_tiles(dtype, hd, S):
    """8, 16 and 128 query rows a KV head and one more, on rows of several pages, an idle one and one that is all new."""
    lens, counts = [300, S, 90 + S, 64], [S, S, max(1, S - 3), 0]
    c, ks, vs = _filled(4, lens, counts, 2, hd, seed=S)
    q = _rand((4, S, 8, hd), dtype, 5, 1.5)
    _check_attend(c.attend(0, q.cuda()), q, ks, vs, lens, counts, hd ** -0.5)
    _check_attend(c.attend(0, q.cuda(), sliding_window=70), q, ks, vs, lens, counts, hd ** -0.5, 70)


def test_float32_keeps_its_digits_over_a_long_row():
    """The maximum of a long row moves many times, and its terms are summed thousands at a time: the results stay as near to
    64 bits as float32 sums of 8000 terms in blocks of 16 are, whatever the order of the keys."""
    n, hd, heads = 8000, 128, 8
    for rows, scale in ((1, hd ** -0.5), (40, hd ** -0.5), (40, 4 * hd ** -0.5)):
        c, ks, vs = _filled(1, [n], [rows], 2, hd, seed=7)
        m = n
        q = _rand((1, rows, heads, hd), torch.float32, 5)
        got = c.attend(0, q.cuda(), scale=scale)[0].double().cpu()
        k, v = ks[0][:m], vs[0][:m]
        want = K.attend(q[0].double(), k, v, m, rows, scale, 0)
        # float32 roundings (2^-24 each): a score is 4 group sums of 32 products in three parts, rounded to within 2^-22 of
        # the sum of its magnitudes; its exponent, and the maximum's, to 2^-24 of themselves (2^-23 after both); 2^x to
        # 2^-22; the rows' sums grow over 500 blocks, each to 2^-24 of what is there
        big = torch.einsum("shd,thd->sht", q[0].double().abs(), k.abs().repeat_interleave(heads // 2, 1)).amax(-1) * scale
        A = K.attend(q[0].double(), k, v.abs(), m, rows, scale, 0)
        tol = A * (2 * (big[..., None] * (2.0 ** -22 + 2.0 ** -23) + 2.0 ** -22) + 500 * 2.0 ** -24)
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()
        # the roundings are as often up as down: the root mean square stays near the largest kind, that of an exponent of
        # magnitude up to 16 (at a scale of hd^-0.5; four times that at four times the scale)
        rms = float((got - want).pow(2).mean().sqrt() / want.pow(2).mean().sqrt())
        assert rms <= 16 * 2.0 ** -24 * max(1.0, scale * hd ** 0.5), rms


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,heads,rows,S", [(256, 8, 8, 70), (128, 8, 3, 701), (64, 3, 40, 140)])
@pytest.mark.parametrize("before", [0, 1, 2, 63])
def test_large_appends_are_exact(dtype, hd, heads, rows, S, before):
    """Calls of many tokens go in tiles of four positions: rows that begin and end anywhere in a tile, special groups."""
    width = -(-(before + S) // PAGE)
    c = _cache(1, rows * width, rows, width * PAGE, heads, hd, fill=0xA5)
    if before:
        c.extend(before)
        c.append(0, torch.ones(rows, before, heads, hd, dtype=dtype, device="cuda"),
                 torch.ones(rows, before, heads, hd, dtype=dtype, device="cuda"))
    counts = [S if r % 3 == 0 else max(0, S - 5 * r - 1) for r in range(rows)]
    k, v = _rand((rows, S, heads, hd), dtype, 1, 3.0), _rand((rows, S, heads, hd), dtype, 2, 1e-3)
    k[:, 3::7, 0] *= 1e-33                                 # scales below and above the quick division's range
    k[:, 4::7, 0] *= 1e33
    k[:, 5::7, 0] = 0.0
    v[:, 2::9, -1, 7], v[:, 3::9, -1, 40] = float("nan"), float("-inf")
    steps = (torch.arange(-15, 17, dtype=torch.float32) * 0.5).clamp(-7, 7)     # every half step, of every scale M / 8
    for i in range(8):
        k[:, 8 + i, 0, :32] = (steps * (8 + i) / 8).to(dtype)
    for r in range(rows):
        k[r, counts[r]:], v[r, counts[r]:] = float("nan"), float("inf")
    c.extend(torch.tensor(counts, dtype=torch.int32, device="cuda"))
    c.append(0, k.cuda(), v.cuda())
    c.check()
    for out in (torch.float32, torch.bfloat16):
        for x, got in zip((k, v), c.read(0, before, S + 3, dtype=out)):
            got = got.double().cpu()
            for r in range(rows):
                want = K.dequantised(x[r, :counts[r]])
                assert torch.equal(torch.isnan(got[r, :counts[r]]), torch.isnan(want))
                assert torch.equal(got[r, :counts[r]].nan_to_num(0), want.nan_to_num(0)), (r, out)
                assert (got[r, counts[r]:] == 0).all()
    if before:
        one = K.dequantised(torch.ones(32, dtype=dtype))[0]
        assert all((x == one.float()).all() for x in c.read(0, 0, before, dtype=torch.float32))


@pytest.mark.parametrize("rows,hd", [(60, 64), (70, 128), (66, 256)])
def test_many_short_chunks(rows, hd):
    """Enough rows of a few queries that they share the tiles of 128, several (row, KV head) to a CTA: ragged counts, idle
    and empty rows, one page and two."""
    rng = random.Random(rows)
    S, kv, heads = 9, 4, 8
    counts = [rng.choice([0, 1, 5, 9, 9]) for _ in range(rows)]
    lens = [n + rng.choice([0, 0, 3, 55, 60, 64]) for n in counts]
    c, ks, vs = _filled(rows, lens, counts, kv, hd, seed=rows)
    q = _rand((rows, S, heads, hd), torch.bfloat16, 5, 1.5)
    for r, n in enumerate(counts):
        q[r, n:] = float("nan")
    for window in (0, 7):
        got = c.attend(0, q.cuda(), sliding_window=window or None)
        _check_attend(got, q, ks, vs, lens, counts, hd ** -0.5, window)
    c.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,kv,hd,S,room", [(2, 2, 64, 70, 500), (2, 2, 128, 70, 500), (3, 1, 256, 40, 500), (2, 2, 128, 70, 0),
                                               (90, 4, 64, 9, 0), (90, 4, 128, 9, 500), (4, 2, 64, 3, 0), (4, 2, 64, 3, 500)])
def test_padding_is_zero_beside_a_nan(dtype, rows, kv, hd, S, room):
    """Queries behind a row's counts are zeros also where a key or value that lies whole pages before the chunk decodes to
    NaN and the tile's other queries see it."""
    heads, before = 2 * kv, 200
    counts = [max(0, S - 1 - r % S) for r in range(rows)]
    width = -(-(before + S) // PAGE)
    c = _cache(1, rows * width, rows, (width + room) * PAGE, kv, hd)
    k, v = _rand((rows, before, kv, hd), torch.float32, 1), _rand((rows, before, kv, hd), torch.float32, 2)
    k[:, 5, 0, 3] = float("nan")
    v[:, 150, kv - 1, 40] = float("inf")
    c.extend(before)
    c.append(0, k.cuda(), v.cuda())
    c.extend(torch.tensor(counts, dtype=torch.int32, device="cuda"))
    x = _rand((rows, S, kv, hd), torch.float32, 3).cuda()
    c.append(0, x, x)
    q = _rand((rows, S, heads, hd), dtype, 4).cuda()
    for window in (None, 190):
        got = c.attend(0, q, sliding_window=window).cpu()
        sees = window is None
        for r, n in enumerate(counts):
            assert (got[r, n:] == 0).all(), (r, n)
            first, last = got[r, :n, :2], got[r, :n, -2:]
            if sees:
                assert torch.isnan(first).all()
            assert torch.isnan(last[..., 32:64]).all() and (kv == 1 or torch.isfinite(last[..., :32]).all())
    c.check()


@pytest.mark.parametrize("how", ["an earlier error", "no room", "a layer raises"])
def test_a_model_call_that_fails_leaves_the_rows(how, monkeypatch):
    """What apply raises over a paged cache, it raises with the rows as they were: an error that an earlier call left on the
    device, a pool that is full, a layer that fails half way."""
    from jaxml_b200 import PagedKVCache, decoders

    model, params = _tiny("llama")
    cfg = model.config
    ids = torch.randint(0, cfg.vocab_size, (2, 70), generator=torch.Generator().manual_seed(0), dtype=torch.int32)
    new = lambda: PagedKVCache.init(cfg.num_layers, 6, 2, 256, cfg.num_key_value_heads, 64)  # noqa: E731
    c, want = new(), new()
    for x in (c, want):
        model.apply(params, ids, kv_caches=x)
    state = [t.clone() for t in (c.table, c.lengths, c.refs)]
    if how == "an earlier error":
        c.rollback(10 ** 6)
        with pytest.raises(RuntimeError, match="device status"):
            model.apply(params, ids[:, :60], kv_caches=c)
    elif how == "no room":
        with pytest.raises(RuntimeError, match="no room"):
            model.apply(params, torch.cat([ids, ids], 1), kv_caches=c)
    else:
        real = decoders.layered_forward

        def half(family, cfg, *args, **kw):
            real(family, cfg, *args, **kw)
            raise OSError("a layer")

        monkeypatch.setattr(decoders, "layered_forward", half)
        with pytest.raises(OSError, match="a layer"):
            model.apply(params, ids[:, :60], kv_caches=c)
        monkeypatch.setattr(decoders, "layered_forward", real)
    assert all(torch.equal(a, b) for a, b in zip(state, (c.table, c.lengths, c.refs)))
    a, b = (model.apply(params, ids[:, :60], kv_caches=x).logits for x in (c, want))
    assert torch.equal(a, b) and c.lengths.tolist() == [130, 130]


def test_the_caches_own_lengths_and_counts_as_arguments():
    """extend and rollback by the lengths or counts of the cache itself are what they are by a copy of them."""
    rows = 40
    lens = [(37 * r) % 150 for r in range(rows)]

    def new():
        c = _cache(1, 8 * rows, rows, 10 * PAGE, 1, 64)
        c.extend(lens)
        c.fork([r - r % 3 for r in range(rows)])          # shared last pages
        c.extend([r % 4 for r in range(rows)])
        return c

    for name in ("lengths", "counts"):
        for call in ("extend", "rollback"):
            a, b = new(), new()
            getattr(a, call)(getattr(a, name))
            getattr(b, call)(getattr(b, name).clone())
            a.check()
            b.check()
            assert all(torch.equal(getattr(a, x), getattr(b, x)) for x in ("table", "lengths", "counts", "refs")), (name, call)
            with pytest.raises(RuntimeError, match="own state"):
                a.fork(getattr(a, name))


@pytest.mark.parametrize("length", [4 * PAGE + 1, 2 ** 31 - 64, 2 ** 31 - 62, 2 ** 31 - 1, -1, -2 ** 31])
def test_lengths_that_no_row_can_have(length):
    """A cache made of given tensors may hold anything: such a row is reported, nothing out of range is touched, and free
    empties it where its length is positive."""
    c, ks, vs = _filled(3, [100, 200, 256], [1, 1, 1], 2, 64, seed=4)
    assert c.row_pages == 4
    c.lengths[1] = length
    q = _rand((3, 1, 4, 64), torch.bfloat16, 5).cuda()
    table, refs = c.table.clone(), c.refs.clone()
    assert torch.isfinite(c.attend(0, q)[[0, 2]]).all()
    c.append(0, q[:, :, :2], q[:, :, :2])
    assert (c.read(0, 300, 8)[0] == 0).all()
    c.status.zero_()
    for call in (lambda: c.extend(1), lambda: c.rollback([0, 1, 0]), lambda: c.rollback([0, 70, 0]), lambda: c.rollback([0, -1, 0])):
        call()
        with pytest.raises(RuntimeError, match="device status 4"):
            c.check()
        assert torch.equal(c.table, table) and torch.equal(c.refs, refs)
        assert c.lengths.tolist() == [100, length, 256] and c.counts[1] == 0
    c.free([1])
    if length > 0:
        c.check()
        assert c.lengths.tolist() == [100, 0, 256] and (c.table[1] == -1).all() and int(c.refs.sum()) == 6


def test_a_mask_that_disagrees_with_the_counts_is_refused():
    """A block over a layer of the cache takes the call's tokens from its counts: a mask may say the same, nothing else."""
    from jaxml_b200 import ModelConfig
    from jaxml_b200.nn import Attention

    cfg = ModelConfig(head_dim=64, hidden_size=256, num_heads=4, num_kv_heads=2, num_layers=1, max_position_embeddings=256,
                      vocab_size=512)
    block = Attention(cfg, dtype=torch.float32)
    x = _rand((2, 5, 256), torch.float32, 1).cuda()
    variables = block.init(0, x)
    c = _cache(1, 4, 2, 128, 2, 64)
    c.extend([5, 3])
    pages = c.pages.clone()
    for bad in (torch.ones(2, 5, dtype=torch.bool), torch.tensor([[1, 1, 1, 1, 1], [1, 1, 0, 0, 0]]).cuda()):
        with pytest.raises(ValueError, match="attention_mask must hold the cache's counts"):
            block.apply(variables, x, attention_mask=bad, kv_cache=c.layer(0))
    assert torch.equal(c.pages, pages)
    mask = torch.tensor([[1, 1, 1, 1, 1], [1, 1, 1, 0, 0]])
    a = block.apply(variables, x, attention_mask=mask, kv_cache=c.layer(0)).attention_output
    b = block.apply(variables, x, kv_cache=c.layer(0)).attention_output
    assert torch.equal(a, b)


@pytest.mark.parametrize("rows,hd", [(80, 64), (130, 64), (100, 256)])
def test_many_short_chunks_in_tiles_of_128(rows, hd):
    """More (row, query tile, KV head) segments than groups are taken for (512), so that several of them come to a CTA of the
    kernel for tiles of 128 rows at every head size."""
    rng = random.Random(rows)
    S, kv, heads = 9, 4, 8
    assert rows * -(-S * heads // kv // 16) * kv > 512
    counts = [rng.choice([0, 1, 5, 9, 9]) for _ in range(rows)]
    lens = [n + rng.choice([0, 0, 3, 55, 60, 64, 200]) for n in counts]
    c, ks, vs = _filled(rows, lens, counts, kv, hd, seed=rows)
    q = _rand((rows, S, heads, hd), torch.bfloat16, 5, 1.5)
    for r, n in enumerate(counts):
        q[r, n:] = float("nan")
    for window in (0, 7):
        got = c.attend(0, q.cuda(), sliding_window=window or None)
        _check_attend(got, q, ks, vs, lens, counts, hd ** -0.5, window)
    c.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_pool_of_more_than_32_bits(dtype):
    """Pages that lie more than 2^32 bytes into the pool: written, read, attended to by each kernel, copied on a write."""
    heads, hd, layers, pages = 8, 256, 2, 20000
    c = _cache(layers, pages, 2, 600 * PAGE, heads, hd)
    assert c.pages.numel() > 2 ** 32 + 2 ** 30
    c.refs[:pages - 40] = 1                     # held by others: the rows' pages are the last ones
    n = [150, 130]
    k, v = _rand((2, max(n), heads, hd), dtype, 1), _rand((2, max(n), heads, hd), dtype, 2)
    c.extend(n)
    c.append(layers - 1, k.cuda(), v.cuda())
    c.check()
    assert int(c.table[c.table >= 0].min()) >= pages - 40
    for x, got in zip((k, v), c.read(layers - 1, 0, max(n), dtype=torch.float32)):
        for r in range(2):
            assert torch.equal(got[r, :n[r]].double().cpu(), K.dequantised(x[r, :n[r]]))
    ks, vs = _Rows([k[r, :n[r]] for r in range(2)]), _Rows([v[r, :n[r]] for r in range(2)])
    last = _rand((2, max(n), heads, hd), dtype, 3)
    _check_attend(c.attend(layers - 1, last.cuda()), last, ks, vs, n, n, hd ** -0.5)
    c.rollback(1)
    c.extend(1)
    c.append(layers - 1, *(torch.stack([x[r, n[r] - 1:n[r]] for r in range(2)]).cuda() for x in (k, v)))
    q = _rand((2, 1, 2 * heads, hd), dtype, 4)
    _check_attend(c.attend(layers - 1, q.cuda()), q, ks, vs, n, [1, 1], hd ** -0.5)
    _check_attend(c.attend(layers - 1, q.cuda(), sliding_window=100), q, ks, vs, n, [1, 1], hd ** -0.5, 100)
    before = c.read(layers - 1, 0, n[0])[0][0]
    c.fork([0, 0])
    c.extend(1)
    c.append(layers - 1, torch.zeros(2, 1, heads, hd, dtype=dtype, device="cuda"),
             torch.zeros(2, 1, heads, hd, dtype=dtype, device="cuda"))
    c.check()
    assert c.table[0, 2] != c.table[1, 2]
    got = c.read(layers - 1, 0, n[0] + 1)[0]
    assert all(torch.equal(got[r, :n[0]], before) and (got[r, n[0]] == 0).all() for r in range(2))


def test_a_captured_change_of_rows_gives_the_eager_results():
    """free, compact, extend, append and attend in one graph: each replay frees and admits the rows that its inputs name."""
    def state():
        c = _cache(2, 40, 4, 300, 2, 64, fill=0xFF)
        c.extend([60, 3, 200, 130])
        x = _rand((4, 200, 2, 64), torch.bfloat16, 1).cuda()
        for layer in range(2):
            c.append(layer, x, x)
        return c

    def turn(c, gone, admit, kv, q):
        c.free(gone)
        used = c.compact()
        c.extend(admit)
        c.append(1, kv, kv)
        return used, c.attend(1, q)

    gone, admit = torch.zeros(4, dtype=torch.bool, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    kv, q = torch.zeros(4, 70, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 70, 4, 64, dtype=torch.bfloat16, device="cuda")
    a, b = state(), state()
    turn(b, gone, admit, kv, q)                 # loads what is loaded once
    b = state()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = turn(b, gone, admit, kv, q)
    for i in range(8):
        gone.copy_(torch.tensor([(i + r) % 3 == 0 for r in range(4)]))
        admit.copy_(torch.tensor([70 if (i + r) % 3 == 0 else 1 for r in range(4)]))
        kv.copy_(_rand((4, 70, 2, 64), torch.bfloat16, 10 + i))
        q.copy_(_rand((4, 70, 4, 64), torch.bfloat16, 40 + i))
        want = turn(a, gone, admit, kv, q)
        graph.replay()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
        assert all(torch.equal(getattr(a, x), getattr(b, x)) for x in ("table", "lengths", "counts", "refs")), i
    a.check()
    b.check()
