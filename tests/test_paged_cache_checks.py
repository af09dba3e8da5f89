"""The paged 4-bit cache and token scoring without a GPU: argument checks, refusals of the C entries, and the properties
of the number format and of the page management that the device tests rely on."""
import ctypes
import random

import numpy as np
import pytest
import torch

from jaxml_b200 import PagedKVCache
from jaxml_b200 import _native as N
from jaxml_b200.paged_cache import block_bytes
from jaxml_b200.sampling import token_log_probs
from oracle import kv4_oracle as K


def _cpu_cache(rows=2, n_pages=4, row_pages=3, heads=2, hd=64, layers=1, **over):
    t = dict(pages=torch.zeros(layers, n_pages, heads, block_bytes(hd), dtype=torch.uint8),
             table=torch.full((rows, row_pages), -1, dtype=torch.int32), lengths=torch.zeros(rows, dtype=torch.int32),
             counts=torch.zeros(rows, dtype=torch.int32), refs=torch.zeros(n_pages, dtype=torch.int32), head_dim=hd)
    t.update(over)
    return PagedKVCache(**t)


def test_constructor_refusals():
    _cpu_cache()
    with pytest.raises(NotImplementedError, match="head_dim of 64, 128 or 256"):
        _cpu_cache(hd=96)
    with pytest.raises(TypeError, match="lengths must be a 1D"):
        _cpu_cache(lengths=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="one entry per row"):
        _cpu_cache(counts=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="one entry per page"):
        _cpu_cache(refs=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="blocks of"):
        _cpu_cache(pages=torch.zeros(1, 4, 2, 100, dtype=torch.uint8))
    with pytest.raises(ValueError, match="contiguous"):
        _cpu_cache(table=torch.full((3, 2), -1, dtype=torch.int32).T)
    with pytest.raises(ValueError, match="at most 8192 rows"):
        _cpu_cache(rows=8193)
    with pytest.raises(RuntimeError, match="CUDA device"):
        PagedKVCache.init(1, 4, 2, 64, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="num_pages must be positive"):
        PagedKVCache.init(1, 0, 2, 64, 2, 64)
    with pytest.raises(TypeError, match="num_rows must be an integer"):
        PagedKVCache.init(1, 4, 2.0, 64, 2, 64)


def test_call_refusals():
    c = _cpu_cache()
    kv = torch.zeros(2, 1, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA device"):
        c.append(0, kv, kv)
    with pytest.raises(ValueError, match="layer must be within"):
        c.append(1, kv, kv)
    with pytest.raises(TypeError, match="layer must be an integer"):
        c.append(0.0, kv, kv)
    with pytest.raises(ValueError, match="k must have shape"):
        c.append(0, kv[:1], kv)
    with pytest.raises(TypeError, match="v must be float32 or bfloat16"):
        c.append(0, kv, kv.half())
    with pytest.raises(ValueError, match="same shape and dtype"):
        c.append(0, kv, torch.zeros(2, 2, 2, 64))
    with pytest.raises(ValueError, match="empty axes"):
        c.append(0, kv[:, :0], kv[:, :0])
    with pytest.raises(ValueError, match="multiple of the 2 KV heads"):
        c.attend(0, torch.zeros(2, 1, 3, 64))
    with pytest.raises(ValueError, match="sliding_window must be positive"):
        c.attend(0, torch.zeros(2, 1, 4, 64), sliding_window=0)
    with pytest.raises(ValueError, match="scale must be finite"):
        c.attend(0, torch.zeros(2, 1, 4, 64), scale=float("nan"))
    with pytest.raises(ValueError, match="counts must not be negative"):
        c.extend(-1)
    with pytest.raises(ValueError, match="counts must have shape"):
        c.extend([1, 2, 3])
    with pytest.raises(TypeError, match="counts must contain integers"):
        c.extend([1.0, 2.0])
    with pytest.raises(ValueError, match="parents must have shape"):
        c.fork([0])
    with pytest.raises(ValueError, match="n must not be negative"):
        c.rollback(-1)
    with pytest.raises(ValueError, match="boolean tensor"):
        c.free(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="rows must be within"):
        c.free([2])
    with pytest.raises(TypeError, match="dtype must be float32 or bfloat16"):
        c.read(0, dtype=torch.float16)
    with pytest.raises(ValueError, match="length must be positive"):
        c.read(0, 0, 0)
    with pytest.raises(ValueError, match="num_pages must be positive"):
        c.resize(0)


def test_resize_refuses_to_drop_used_pages():
    c = _cpu_cache(refs=torch.tensor([0, 0, 0, 1], dtype=torch.int32))
    with pytest.raises(ValueError, match="below a used page"):
        c.resize(3)
    d = c.resize(6)
    assert d.num_pages == 6 and d.refs.tolist() == [0, 0, 0, 1, 0, 0]


def _native_cache(**over):
    v = dict(pages=1 << 12, table=1 << 12, lengths=1 << 12, counts=1 << 12, refs=1 << 12, status=1 << 12, num_layers=1,
             num_pages=4, num_rows=2, row_pages=3, num_kv_heads=2, head_dim=64)
    v.update(over)
    c = N.JxKv4Cache()
    for name, x in v.items():
        setattr(c, name, x)
    return c


@pytest.mark.parametrize("over,code", [(dict(pages=None), N.JX_ERR_ARG), (dict(refs=None), N.JX_ERR_ARG),
                                       (dict(pages=(1 << 12) + 8), N.JX_ERR_ARG), (dict(num_rows=0), N.JX_ERR_SHAPE),
                                       (dict(num_rows=8193), N.JX_ERR_SHAPE), (dict(head_dim=96), N.JX_ERR_SHAPE),
                                       (dict(row_pages=(1 << 24) + 1), N.JX_ERR_SHAPE), (dict(num_kv_heads=0), N.JX_ERR_SHAPE)])
def test_c_entries_refuse_a_bad_cache(over, code):
    lib, c, p = N.load(), _native_cache(**over), 1 << 12
    ints, size = N.LL(), N.LL()
    assert lib.jx_kv4_append(c, 0, 1, p, 1, 1, 1, p, 1, 1, 1, N.JX_BF16, None) == code
    assert lib.jx_kv4_read(c, 0, None, 0, 1, p, p, N.JX_BF16, None) == code
    assert lib.jx_kv4_attend(c, 0, 1, 2, p, 1, 1, 1, p, 1.0, 0, p, 1 << 40, N.JX_BF16, None) == code
    assert lib.jx_kv4_attend_workspace(c, 1, 2, N.JX_BF16, size) == code
    assert lib.jx_kv4_workspace_ints(c, ints) == code
    assert lib.jx_kv4_extend(c, None, 1, p, 1 << 40, None) == code
    assert lib.jx_kv4_fork(c, p, None) == code
    assert lib.jx_kv4_rollback(c, None, 1, None) == code
    assert lib.jx_kv4_free(c, p, None) == code
    assert lib.jx_kv4_compact(c, p, p, 1 << 40, None) == code


def test_c_entries_refuse_bad_arguments():
    lib, c, p = N.load(), _native_cache(), 1 << 12
    A, S, D = N.JX_ERR_ARG, N.JX_ERR_SHAPE, N.JX_ERR_DTYPE
    app = lambda layer=0, S_=1, k=p, v=p, dt=N.JX_BF16: lib.jx_kv4_append(c, layer, S_, k, 1, 1, 1, v, 1, 1, 1, dt, None)  # noqa: E731
    assert [app(layer=1), app(layer=-1), app(S_=0)] == [S] * 3
    assert [app(k=None), app(v=p + 1), app(k=p + 2, dt=N.JX_F32)] == [A] * 3 and app(dt=7) == D
    rd = lambda layer=0, n=1, k=p, dt=N.JX_BF16: lib.jx_kv4_read(c, layer, None, 0, n, k, p, dt, None)  # noqa: E731
    assert [rd(layer=1), rd(n=0)] == [S] * 2 and [rd(k=None), rd(k=p + 8)] == [A] * 2 and rd(dt=3) == D
    size = N.LL()
    assert lib.jx_kv4_attend_workspace(c, 1, 4, N.JX_BF16, size) == N.JX_OK and size.value == 0     # short tables need none
    long = _native_cache(row_pages=1000)
    assert lib.jx_kv4_attend_workspace(long, 1, 4, N.JX_BF16, size) == N.JX_OK and size.value > 0
    assert lib.jx_kv4_attend(long, 0, 1, 4, p, 1, 1, 1, p, 1.0, 0, p, size.value - 1, N.JX_BF16, None) == A
    assert lib.jx_kv4_attend(long, 0, 1, 4, p, 1, 1, 1, p, 1.0, 0, None, 1 << 40, N.JX_BF16, None) == A
    assert lib.jx_kv4_attend_workspace(c, 0, 4, N.JX_BF16, size) == S
    assert lib.jx_kv4_attend_workspace(c, 1, 3, N.JX_BF16, size) == S

    def att(layer=0, S_=1, Hq=4, q=p, out=p, scale=1.0, window=0, ws=p, n=1 << 40, dt=N.JX_BF16):
        return lib.jx_kv4_attend(c, layer, S_, Hq, q, 1, 1, 1, out, scale, window, ws, n, dt, None)

    assert [att(layer=1), att(S_=0), att(Hq=3), att(Hq=0), att(window=-1), att(S_=1 << 30)] == [S] * 6
    assert [att(q=None), att(q=p + 1), att(out=p + 2), att(ws=p + 8), att(scale=float("nan"))] == [A] * 5
    assert att(dt=2) == D
    assert lib.jx_kv4_extend(c, None, -1, p, 1 << 40, None) == S
    assert lib.jx_kv4_extend(c, None, 1, None, 1 << 40, None) == A and lib.jx_kv4_extend(c, None, 1, p, 3, None) == A
    assert lib.jx_kv4_fork(c, None, None) == A and lib.jx_kv4_free(c, None, None) == A
    assert lib.jx_kv4_rollback(c, None, -1, None) == S
    assert lib.jx_kv4_compact(c, None, p, 1 << 40, None) == A and lib.jx_kv4_compact(c, p, p, 0, None) == A


def test_scoring_refusals():
    with pytest.raises(RuntimeError, match="CUDA logits only"):
        token_log_probs(torch.zeros(2, 5), [0, 1])
    lib, p = N.load(), 1 << 12

    def rc(**over):
        v = dict(rows=2, V=100, logits=p, ld=100, dtype=N.JX_F32, top_n=3, ids=p, log_probs=p, entropy=p, top_log_probs=p,
                 top_ids=p)
        v.update(over)
        a = N.JxLogProbsArgs()
        for name, x in v.items():
            setattr(a, name, x)
        return lib.jx_token_log_probs(a, None)

    assert [rc(logits=None), rc(ids=None), rc(entropy=None), rc(top_ids=None), rc(logits=p + 2)] == [N.JX_ERR_ARG] * 5
    assert [rc(rows=0), rc(V=0), rc(ld=99), rc(top_n=-1), rc(top_n=65), rc(V=2, ld=2)] == [N.JX_ERR_SHAPE] * 6
    assert rc(dtype=5) == N.JX_ERR_DTYPE
    assert lib.jx_token_log_probs(None, None) == N.JX_ERR_ARG


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import shutil
    import subprocess

    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    inc = os.path.join(os.path.dirname(N.__file__), os.pardir, "include")
    pairs = [(N.JxKv4Cache, "jx_kv4_cache"), (N.JxLogProbsArgs, "jx_log_probs_args")]
    body = "".join(f'printf("{n} sizeof %zu\\n", sizeof({n}));' +
                   "".join(f'printf("{n} {f} %zu\\n", offsetof({n}, {f}));' for f, _ in c._fields_) for c, n in pairs)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "jxb200.h"\nint main(void) {' + body + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(exe)], check=True)
    got = {tuple(ln.split()[:2]): int(ln.split()[2]) for ln in
           subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()}
    for cls, name in pairs:
        assert got[(name, "sizeof")] == ctypes.sizeof(cls)
        assert all(got[(name, f)] == getattr(cls, f).offset for f, _ in cls._fields_)


def test_more_positions_than_a_table_holds_are_refused():
    lib, p = N.load(), 1 << 20
    c = _native_cache()
    for n in ((1 << 30) + 1, 2 ** 31 - 1):
        assert lib.jx_kv4_append(c, 0, n, p, 0, 0, 1, p, 0, 0, 1, N.JX_BF16, None) == N.JX_ERR_SHAPE
        assert lib.jx_kv4_read(c, 0, None, 0, n, p, p, N.JX_BF16, None) == N.JX_ERR_SHAPE


# -- the format -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [1e-39, 1e-30, 1e-3, 1.0, 1e4, 1e30])
def test_values_are_exact_in_bfloat16_and_within_half_a_step(scale):
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(300, 64, generator=g, dtype=torch.float64) * scale).float()
    n, s = K.quantise(x)
    v = K.value(n, s)
    assert torch.equal(v.to(torch.bfloat16).double(), v)
    assert torch.equal(s.to(torch.bfloat16).double(), s)
    step = s.repeat_interleave(32, -1)
    live = step > 2.0 ** -126             # below it a scale has fewer significant bits
    assert ((v - x.double()).abs() <= step / 2 * (1 + 1e-12))[live].all()
    # a scale is a multiple of 2^-129, the spacing of 4 significant bits at 2^-126: 3e-39 / 7 rounds to none of it
    assert n.abs().max() == (7 if scale > 1e-38 else 0)


def test_groups_that_are_not_finite_or_too_large_decode_to_nan():
    x = torch.ones(5, 64)
    x[0, 3], x[1, 40], x[2, 5], x[3, 6] = float("nan"), float("inf"), 2.0 ** 122, -2.0 ** 121
    v = K.dequantised(x)
    bad = torch.isnan(v).unflatten(-1, (2, 32)).all(-1)
    assert bad.tolist() == [[True, False], [False, True], [True, False], [False, False], [False, False]]
    assert torch.isnan(v).sum() == 3 * 32


# -- the page management ------------------------------------------------------------------------------------
def test_page_management_keeps_what_rows_wrote():
    """Random calls against rows that each keep their own list: sharing and copying never mix rows."""
    rng = random.Random(0)
    R, P, n = 5, 4, 16
    c, rows, tag = K.Pages(R, P, n), [[] for _ in range(R)], 0
    for _ in range(400):
        what = rng.choice(["extend", "extend", "fork", "rollback", "free", "compact"])
        if what == "extend":
            counts = [rng.choice([0, 1, 3, 64, 70]) for _ in range(R)]
            c.extend(counts)
            for r in range(R):
                for i in range(c.counts[r]):
                    tag += 1
                    c.write(r, c.lengths[r] - c.counts[r] + i, tag)
                    rows[r].append(tag)
        elif what == "fork":
            parents = [rng.randrange(-1, R) for _ in range(R)]
            c.fork(parents)
            rows = [[] if p < 0 else list(rows[p]) for p in parents]
        elif what == "rollback":
            cut = [rng.randrange(0, len(x) + 1) if rng.random() < 0.5 else 0 for x in rows]
            c.rollback(cut)
            rows = [x[:len(x) - k] for x, k in zip(rows, cut)]
        elif what == "free":
            gone = [r for r in range(R) if rng.random() < 0.3]
            c.free(gone)
            rows = [[] if r in gone else x for r, x in enumerate(rows)]
        else:
            used = c.compact()
            assert all(p < used for t in c.table for p in t)
        assert [c.row(r) for r in range(R)] == rows


def test_row_vectors_in_the_caches_own_state_are_refused():
    """A call changes the table, the lengths, the counts and the holders while it reads its row vector."""
    lib, A = N.load(), N.JX_ERR_ARG
    at = dict(table=0x10000, lengths=0x20000, counts=0x30000, refs=0x40000, status=0x50000)
    c = _native_cache(num_rows=8, num_pages=100, row_pages=3, **at)
    inside = [at["table"], at["table"] + 4 * 8 * 3 - 4, at["table"] - 4, at["lengths"] + 4, at["lengths"] - 4, at["counts"] + 28,
              at["refs"], at["refs"] + 396, at["status"], at["status"] - 28]
    for p in inside:
        assert lib.jx_kv4_extend(c, p, 0, 0x60000, 1 << 40, None) == A, hex(p)
        assert lib.jx_kv4_rollback(c, p, 0, None) == A and lib.jx_kv4_fork(c, p, None) == A, hex(p)
    for p in (at["lengths"], at["counts"]):
        assert lib.jx_kv4_fork(c, p, None) == A
    for p in (at["table"] - 7, at["refs"] + 399, at["status"] + 3, at["counts"]):
        assert lib.jx_kv4_free(c, p, None) == A, hex(p)


def test_a_table_of_more_entries_than_32_bits_count_is_refused():
    """Rows could ask for more pages than an int holds, and the plan of an extend would place them outside its list."""
    lib, p, n = N.load(), 1 << 12, N.LL()
    for rows, row_pages in ((8192, 1 << 24), (128, 1 << 24), (8192, 1 << 18)):
        c = _native_cache(num_rows=rows, row_pages=row_pages)
        assert lib.jx_kv4_workspace_ints(c, n) == N.JX_ERR_SHAPE
        assert b"2^31" in lib.jx_last_error()
        assert lib.jx_kv4_extend(c, None, 1, p, 1 << 40, None) == N.JX_ERR_SHAPE
    assert lib.jx_kv4_workspace_ints(_native_cache(num_rows=127, row_pages=1 << 24), n) == N.JX_OK


@pytest.mark.parametrize("dtype,big", [(torch.uint32, 2 ** 32 - 1), (torch.uint32, 2 ** 31), (torch.uint64, 2 ** 64 - 1),
                                       (torch.uint64, 2 ** 63), (torch.uint64, 2 ** 32 + 1), (torch.int64, 2 ** 32 + 1)])
def test_unsigned_row_vectors_do_not_wrap(dtype, big):
    """A parent of 2^32 - 1 is out of range; narrowed bit by bit it would be -1, which empties the row."""
    t = torch.from_numpy(np.array([big, 1], dtype=str(dtype).split(".")[1]))
    assert t.dtype == dtype and _cpu_cache()._row_ints("parents", t).tolist() == [2 ** 31 - 1, 1]
    small = torch.tensor([3, 1]).to(dtype)
    assert _cpu_cache()._row_ints("parents", small).tolist() == [3, 1]


def test_numpy_row_vectors_are_taken_as_lists_are():
    c = _cpu_cache()
    for call in (c.extend, c.rollback, c.fork, lambda x: c.read(0, x, 1)):
        for x in ([1, 0], np.array([1, 0]), np.array([1, 0], dtype=np.int16)):
            with pytest.raises(RuntimeError, match="CUDA device"):      # past its checks
                call(x)
        with pytest.raises(ValueError, match="must have shape"):
            call(np.array([1, 0, 2]))
        with pytest.raises(TypeError, match="must contain integers"):
            call(np.array([1.0, 0.0]))
    for x in (np.int64(1), 1):
        with pytest.raises(RuntimeError, match="CUDA device"):
            c.extend(x)


def test_pages_that_are_no_tensor_are_refused():
    for pages in (None, np.zeros((1, 4, 2, block_bytes(64)), dtype=np.uint8)):
        with pytest.raises(TypeError, match="pages must be a 4D torch.uint8 tensor"):
            _cpu_cache(pages=pages)
