"""token_log_probs on the GPU against 64-bit sums.

Tolerances.  exp in float32 is off by at most 2 units (2^-22), and a sum of V terms none of whose partial chains is longer
than V / 128 + 64 terms by at most that many roundings of 2^-24, all of positive terms; so log z is off by at most
t = 2^-22 + (V / 128 + 64) 2^-24, and a log probability by t plus 2^-22 of its magnitude (two subtractions, one logarithm).
The entropy adds the same relative error of sum p |d|, d the distance to the maximum.  The alternatives are exact.
"""
import math

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as K

pytestmark = pytest.mark.gpu


def _run(x, ids, top_n):
    from jaxml_b200.sampling import token_log_probs

    return token_log_probs(x, ids, top_n=top_n)


def _check(x, ids, top_n, got):
    """Against float64 torch on the CPU: rows [N, V]."""
    lp, ent, top_lp, top_ids = (t.cpu() for t in got)
    x = x.cpu().double()
    N, V = x.shape
    assert lp.dtype == ent.dtype == top_lp.dtype == torch.float32 and top_ids.dtype == torch.int32
    assert lp.shape == ent.shape == (N,) and top_lp.shape == top_ids.shape == (N, top_n)
    fine = torch.isfinite(x.amax(-1)) & ~torch.isnan(x).any(-1)
    assert torch.isnan(ent[~fine]).all() and torch.isnan(lp[~fine & (ids.cpu() >= 0)]).all()
    ref = torch.log_softmax(x, -1)
    assert (top_ids[torch.isnan(x).any(-1)] == -1).all() and torch.isnan(top_lp[~fine]).all()
    t = 2.0 ** -22 + (V / 128 + 64) * 2.0 ** -24
    for r in range(N):
        if not fine[r]:
            continue
        i = int(ids[r])
        want = 0.0 if i < 0 else float(ref[r, i]) if i < V else math.nan
        if math.isfinite(want):
            assert abs(float(lp[r]) - want) <= t + 2.0 ** -22 * abs(want), (r, float(lp[r]), want)
        else:
            assert float(lp[r]) == want or (math.isnan(want) and math.isnan(float(lp[r])))
        p = ref[r].exp()
        d = torch.where(p > 0, x[r] - x[r].max(), 0.0)
        we, pd = float(-(p * torch.where(p > 0, ref[r], 0.0)).sum()), float((p * d.abs()).sum())
        assert abs(float(ent[r]) - we) <= 2 * t * (1 + pd) + 2.0 ** -22 * (pd + abs(we)), (r, float(ent[r]), we)
        order = torch.sort(x[r], descending=True, stable=True).indices[:top_n]
        assert top_ids[r].tolist() == order.tolist(), r
        w = ref[r][order]
        ok = torch.where(torch.isfinite(w), (top_lp[r].double() - w).abs() <= t + 2.0 ** -22 * w.abs(), top_lp[r].double() == w)
        assert ok.all(), r


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,V,top_n", [(1, 1, 1), (3, 2, 2), (2, 31, 31), (5, 64, 64), (1, 1000, 0), (7, 50304, 5),
                                       (2, 128256, 64), (17, 128256, 20), (1, 262144, 33), (300, 4099, 8), (3, 65537, 1)])
def test_random_rows(dtype, N, V, top_n):
    g = torch.Generator().manual_seed(V + N)
    x = (torch.randn(N, V, generator=g) * 4).to(dtype)
    ids = torch.randint(0, V, (N,), generator=g, dtype=torch.int32)
    _check(x, ids, top_n, _run(x.cuda(), ids.cuda(), top_n))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [700, 40000])
def test_rows_that_are_hard(dtype, V):
    """Ties, sorted rows both ways, a filter's -inf, one finite entry, large magnitudes, signed zeros, the best entries next
    to each other or one block apart, and rows without an answer."""
    g = torch.Generator().manual_seed(V)
    rows = [torch.zeros(V), torch.linspace(-50, 50, V), torch.linspace(50, -50, V), torch.randn(V, generator=g)]
    rows[3][torch.rand(V, generator=g) < 0.99] = float("-inf")
    r = torch.full((V,), float("-inf")); r[V // 3] = -3.0; rows.append(r)
    rows.append(torch.randn(V, generator=g) * 1e30)
    rows.append(torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0))
    r = torch.randn(V, generator=g); r[100:200] += 50; rows.append(r)
    r = torch.randn(V, generator=g); r[::256] += 50; rows.append(r)
    r = torch.randn(V, generator=g); r[:] = torch.sort(r).values; rows.append(r)
    r = torch.randn(V, generator=g); r[V // 2:] = r.max(); rows.append(r)
    r = torch.randn(V, generator=g); r[5] = float("nan"); rows.append(r)
    rows.append(torch.full((V,), float("-inf")))
    r = torch.randn(V, generator=g); r[V - 1] = float("inf"); rows.append(r)
    rows.append(torch.full((V,), torch.finfo(dtype).min))
    r = torch.full((V,), torch.finfo(dtype).min); r[V - 2] = 1.0; rows.append(r)
    x = torch.stack(rows).to(dtype)
    ids = torch.tensor([(i * 37) % V for i in range(len(rows))], dtype=torch.int32)
    ids[4], ids[1], ids[2], ids[0] = V // 3, -1, V, V - 1
    for top_n in (0, 1, 64):
        _check(x, ids, top_n, _run(x.cuda(), ids.cuda(), top_n))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shapes_strides_and_id_types(dtype):
    g = torch.Generator().manual_seed(0)
    base = (torch.randn(2, 3, 5003, generator=g) * 2).to(dtype)
    ids = torch.randint(0, 4000, (2, 3), generator=g)
    b, want = base.cuda(), None
    for x in (b[..., 1:4001], b[..., 1:4001].contiguous(), b.transpose(0, 1)[..., 1:4001].contiguous().transpose(0, 1),
              b.new_zeros(2, 3, 8000)[..., ::2].copy_(b[..., 1:4001])):
        for i in (ids.to(torch.int32).cuda(), ids, ids.tolist()):
            got = _run(x, i, 7)
            assert got.log_probs.shape == (2, 3) and got.top_ids.shape == (2, 3, 7)
            _check(x.reshape(6, 4000), ids.reshape(6), 7, [t.reshape((6,) + t.shape[2:]) for t in got])
    one = _run(b[0, 0], torch.tensor(5), 2)
    assert one.log_probs.shape == () and one.top_ids.shape == (2,)
    none = _run(b[:0], torch.zeros(0, 3, dtype=torch.int32), 2)
    assert none.top_log_probs.shape == (0, 3, 2)
    wide = _run(b[0, :2], torch.tensor([2 ** 32 + 5, -2 ** 40]), 0)     # not narrowed to other tokens
    assert torch.isnan(wide.log_probs[0]) and wide.log_probs[1] == 0


def test_python_restatement():
    x = torch.tensor([[1.0, 3.0, 3.0, float("-inf"), -2.0]])
    got = _run(x.cuda(), [4], 5)
    lp, ent, top = K.score(x[0], 4, 5)
    assert abs(float(got.log_probs) - lp) < 1e-6 and abs(float(got.entropy) - ent) < 1e-6
    assert got.top_ids[0].tolist() == [i for i, _ in top] == [1, 2, 0, 4, 3]
    assert got.top_log_probs[0, -1] == float("-inf")


def test_refusals():
    x = torch.zeros(2, 10, device="cuda")
    for bad, err, match in (((x, [0], 0), ValueError, "leading shape"), ((x, [0.0, 1.0], 0), TypeError, "integer token ids"),
                            ((x, [0, 1], 11), ValueError, "top_n"), ((x, [0, 1], -1), ValueError, "top_n"),
                            ((x, [0, 1], 1.5), TypeError, "top_n"), ((x.half(), [0, 1], 0), NotImplementedError, "float16"),
                            ((x.long(), [0, 1], 0), TypeError, "floating point"), ((x[:, :0], [0, 1], 0), ValueError, "vocabulary"),
                            ((torch.zeros(2, 100, device="cuda"), [0, 1], 65), ValueError, "top_n")):
        with pytest.raises(err, match=match):
            _run(*bad)


def test_streams_graphs_and_repeats():
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(20, 128256, generator=g) * 4).to(torch.bfloat16).cuda()
    ids = torch.randint(0, 128256, (20,), generator=g, dtype=torch.int32).cuda()
    want = _run(x, ids, 10)
    s, y = torch.cuda.Stream(), x.flip(0).contiguous()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = [_run(y, ids.flip(0), 10) for _ in range(10)]
    same = [_run(x, ids, 10) for _ in range(10)]
    torch.cuda.synchronize()
    for a, b in zip(same, other):
        assert all(torch.equal(p, w) for p, w in zip(a, want)) and all(torch.equal(p.flip(0), w) for p, w in zip(b, want))
    graph, z, zi = torch.cuda.CUDAGraph(), torch.empty_like(x), torch.empty_like(ids)
    with torch.cuda.graph(graph):
        got = _run(z, zi, 10)
    for src, i in ((x, ids), (y, ids.flip(0))):
        z.copy_(src)
        zi.copy_(i)
        graph.replay()
        assert all(torch.equal(p, w) for p, w in zip(got, _run(src, i, 10)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,top_n", [(63, 63), (130, 64), (1003, 17), (5001, 16), (40000, 20), (20011, 0)])
def test_more_rows_than_are_resident(dtype, V, top_n):
    """Above 592 rows a row has fewer threads: random rows, rows full of ties, and rows that are hard, in between."""
    N = 700
    g = torch.Generator().manual_seed(V)
    x = torch.randn(N, V, generator=g) * 4
    x[1::5] = torch.round(x[1::5] * 0.5)                                     # many equal to the last one wanted
    x[2::50], x[3::50] = 0.0, torch.linspace(-50, 50, V)
    x[4::50, V // 2:], x[5::50, : V // 2] = x[4::50].amax(-1, keepdim=True), float("-inf")
    x[6::50, :-1], x[7::50, V // 3], x[8::50, V // 3] = float("-inf"), float("nan"), float("inf")
    x[9::50], x[10::50] = float("-inf"), torch.randn(V, generator=g) * 1e30
    x[11::50, ::128] += 50
    x[12::50, :100] += 50
    x = x.to(dtype)
    ids = torch.randint(-1, V + 1, (N,), generator=g, dtype=torch.int32)
    got = _run(x.cuda(), ids.cuda(), top_n)
    again = _run(x.cuda(), ids.cuda(), top_n)
    assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip(got, again))
    some = torch.cat([torch.arange(0, 100), torch.arange(585, 605), torch.arange(690, 700)])
    _check(x[some], ids[some], top_n, [t.cpu()[some] for t in got])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [1, 700])
@pytest.mark.parametrize("level", [30.0, -100.0, 1000.0, -1000.0, 8000.0, -8000.0])
def test_the_level_of_a_row_does_not_matter(dtype, N, level):
    """A softmax does not change with a constant added to its row: the same tolerance at every level, on random rows and
    on rows with one entry far above the others (log p = 0 there, never above it by more than the tolerance)."""
    V, g = 5003, torch.Generator().manual_seed(int(abs(level)))
    x = torch.randn(N, V, generator=g) * 3 + level
    x[::2, 77] = level + 150
    x = x.to(dtype)
    ids = torch.randint(0, V, (N,), generator=g, dtype=torch.int32)
    ids[::2] = 77
    got = _run(x.cuda(), ids.cuda(), 5)
    some = torch.arange(min(N, 40))
    _check(x[some], ids[some], 5, [t.cpu()[some] for t in got])
    assert (got.log_probs[::2].cpu() <= 2.0 ** -22 + (V / 128 + 64) * 2.0 ** -24).all()


def test_unsigned_ids_do_not_wrap():
    """An id of 2^32 - 1 is beyond the vocabulary (NaN), not the negative id that asks for nothing (0)."""
    x = torch.randn(2, 10, generator=torch.Generator().manual_seed(0)).cuda()
    want = _run(x, [3, 4], 0).log_probs
    for dtype, big in ((np.uint32, 2 ** 32 - 1), (np.uint64, 2 ** 64 - 1), (np.uint64, 2 ** 32 + 3)):
        for dev in ("cpu", "cuda"):
            got = _run(x, torch.from_numpy(np.array([big, 4], dtype=dtype)).to(dev), 0).log_probs
            assert torch.isnan(got[0]) and got[1] == want[1], (dtype, dev)
            assert torch.equal(_run(x, torch.from_numpy(np.array([3, 4], dtype=dtype)).to(dev), 0).log_probs, want)


def test_logits_of_more_than_32_bits():
    """Rows that begin more than 2^31 elements into the logits."""
    N, V = 8300, 262144
    g = torch.Generator().manual_seed(0)
    x = torch.zeros(N, V, dtype=torch.bfloat16, device="cuda")
    some = torch.tensor([0, 1, 4200, 8192, 8298, 8299])
    rows = (torch.randn(len(some), V, generator=g) * 4).to(torch.bfloat16)
    x[some.cuda()] = rows.cuda()
    ids = torch.randint(0, V, (N,), generator=g, dtype=torch.int32)
    got = _run(x, ids.cuda(), 5)
    _check(rows, ids[some], 5, [t.cpu()[some] for t in got])
    flat = torch.ones(N, dtype=torch.bool)
    flat[some] = False
    assert (got.top_ids.cpu()[flat] == torch.arange(5)).all()
    assert (got.log_probs.cpu()[flat] + math.log(V)).abs().max() <= 2.0 ** -22 * (1 + math.log(V)) + (V / 128 + 64) * 2.0 ** -24
