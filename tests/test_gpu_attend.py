"""Attention over the paged cache (ssb_attend_rows) against the plain form in 64 bits; the tolerances are
derived in decoder_plain.py."""
import math

import pytest

import decoder_plain as plain
import speech_sampler as ss

pytestmark = pytest.mark.gpu


def torch_mod():
    import torch
    return torch


def run(engine, c, scale=None, window=0, sinks=0, ragged=True, extra_rows=0, **kw):
    """out and lse of the call, both filled with 7 before; rows behind the last sequence must keep it."""
    torch = torch_mod()
    scale = c.dim ** -0.5 if scale is None else scale
    q = torch.cat([c.q, torch.full((extra_rows, c.heads, c.dim), 3.0, dtype=c.dtype, device="cuda")]) if extra_rows else c.q
    out = torch.full(q.shape, 7.0, dtype=c.dtype, device="cuda")
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    status = torch.full((len(c.lens),), -7, dtype=torch.int32, device="cuda")
    engine.attend(q, c.cache(), c.length, scale, window, sinks, row_start=c.row_start if ragged else None,
                  max_rows=c.max_rows, out=out, lse=lse, status=status, **kw)
    torch.cuda.synchronize()
    assert torch.all(out[c.total:] == 7.0) and torch.all(lse[c.total:] == 7.0)
    return out, lse, status


DTYPES = ["f32", "bf16"]


def dtype_of(name):
    torch = torch_mod()
    return torch.float32 if name == "f32" else torch.bfloat16


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[1], [2, 1, 17], [63, 64, 65], [128, 127, 129, 16], [15, 300, 1000], [2049]])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 1, 64), (8, 4, 128)])
def test_one_token(engine, dtype, lens, heads, kv_heads, dim):
    c = plain.Case(lens, [1] * len(lens), heads, kv_heads, dim, dtype_of(dtype), seed=sum(lens), fill=float("nan"))
    out, lse, status = run(engine, c, ragged=False)
    assert status.tolist() == [ss.ROW_OK] * len(lens)
    plain.check_attend(c, out, lse, dim ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (4, 2), (7, 1), (12, 4), (16, 1), (40, 2), (48, 1)])
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 256])
def test_head_layouts(engine, dtype, heads, kv_heads, dim):
    c = plain.Case([33, 130], [1, 1], heads, kv_heads, dim, dtype_of(dtype), layout="positions", seed=heads + dim)
    out, lse, _ = run(engine, c)
    plain.check_attend(c, out, lse, dim ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["heads", "positions"])
def test_page_sizes(engine, dtype, page, layout):
    c = plain.Case([page - 1, page, page + 1, 3 * page + 5], [1, 2, 1, 3], 4, 2, 128, dtype_of(dtype), page, layout, seed=page,
                   fill=float("inf"))
    out, lse, _ = run(engine, c)
    plain.check_attend(c, out, lse, 128 ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [[2, 5, 1], [5, 0, 3], [9, 16, 17], [33, 1, 64], [65, 40, 129], [200, 3, 257]])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (8, 1, 64)])
def test_drafts_and_prompts(engine, dtype, rows, heads, kv_heads, dim):
    """Rows of one sequence see each other causally; the first sequence is a whole prompt, the others continue one."""
    lens = [rows[0], rows[1] + 70, rows[2] + 301]
    c = plain.Case(lens, rows, heads, kv_heads, dim, dtype_of(dtype), seed=sum(rows), fill=float("nan"))
    out, lse, status = run(engine, c, extra_rows=3)
    assert status.tolist() == [ss.ROW_OK] * 3
    plain.check_attend(c, out, lse, dim ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (65, 64), (100, 130), (128, 65), (300, 4), (5000, 2)])
@pytest.mark.parametrize("rows", [1, 4, 150])
def test_window_and_sinks(engine, dtype, window, sinks, rows):
    lens = [rows, 190 + rows, 700 + rows]
    c = plain.Case(lens, [rows] * 3, 4, 2, 64, dtype_of(dtype), seed=window + rows)
    out, lse, _ = run(engine, c, window=window, sinks=sinks)
    plain.check_attend(c, out, lse, 0.125, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 3, 140])
@pytest.mark.parametrize("page", [16, 128])
def test_pages_behind_a_window_may_be_gone(engine, dtype, rows, page):
    """Entries of pages that no row sees may hold anything, and pages that hold one seen position are read."""
    window, sinks, length = 200, 5, 1501
    c = plain.Case([length, length + 64], [rows, rows], 4, 2, 128, dtype_of(dtype), page, seed=rows)
    for s, n in enumerate(c.lens):
        first = n - rows - window + 1  # the first position that the first row sees
        gone = torch_mod().arange(1, first // page)
        c.table[s, gone] = torch_mod().tensor([-1, 10 ** 9, -2 ** 31], dtype=torch_mod().int32, device="cuda")[gone.cuda() % 3]
    out, lse, status = run(engine, c, window=window, sinks=sinks)
    assert status.tolist() == [ss.ROW_OK] * 2
    for s in range(2):
        c.table[s][(c.table[s] < 0) | (c.table[s] >= len(c.k))] = -1
    plain.check_attend(c, out, lse, 128 ** -0.5, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [4, 150])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_what_a_row_does_not_see_has_no_effect(engine, dtype, rows, value):
    """The newest position's key and value are not finite: the rows before it must not notice, and the last
    must. Under a window, nor must rows past one that has left theirs."""
    torch = torch_mod()
    c = plain.Case([rows + 90, rows + 3], [rows, rows], 4, 2, 128, dtype_of(dtype), seed=rows)
    clean = plain.Case([rows + 90, rows + 3], [rows, rows], 4, 2, 128, dtype_of(dtype), seed=rows)
    window = 40
    for s, n in enumerate(c.lens):
        for p in (n - 1, n - rows - 2):  # seen by the last row alone; seen by the first rows, not by the last ones
            c.v[c.table[s, p // 16].long(), p % 16] = value
            c.k[c.table[s, p // 16].long(), p % 16] = value if math.isnan(value) else 0.25
            clean.k[c.table[s, p // 16].long(), p % 16] = 0.25
    out, lse, _ = run(engine, c, window=window)
    want, want_lse, tol, lse_tol = plain.attend(clean, 128 ** -0.5, window)
    for s, n in enumerate(c.lens):
        base = s * rows
        for i in range(rows):
            p = n - rows + i
            bad = p == n - 1 or p - (n - rows - 2) < window
            if bad:
                assert not torch.isfinite(out[base + i]).any(), (s, i)
            else:
                assert torch.all((out[base + i].double() - want[base + i]).abs() <= tol[base + i]), (s, i)
                assert torch.all((lse[base + i].double() - want_lse[base + i]).abs() <= lse_tol[base + i]), (s, i)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 6, 130])
def test_idle_streams_and_rows(engine, dtype, rows):
    """A stream of length 0, and one with more rows than positions: the rows before position 0 give zeros."""
    lens = [0, 40 + rows, rows - 1, 1]
    c = plain.Case(lens, [rows] * 4, 4, 2, 64, dtype_of(dtype), fill=float("nan"))
    out, lse, status = run(engine, c, ragged=False)
    assert status.tolist() == [ss.ROW_OK] * 4
    assert torch_mod().all(out[:rows] == 0)
    plain.check_attend(c, out, lse, 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 5, 140])
@pytest.mark.parametrize("page_id", [-1, -2 ** 31, 2 ** 31 - 1, "pages"])
def test_bad_pages_refuse_the_sequence(engine, dtype, rows, page_id):
    torch = torch_mod()
    c = plain.Case([300, 400, 350], [rows] * 3, 4, 2, 64, dtype_of(dtype))
    good = c.table.clone()
    c.table[1, 3] = len(c.k) if page_id == "pages" else page_id
    out, lse, status = run(engine, c)
    assert status.tolist() == [ss.ROW_OK, ss.ROW_INVALID_ROW, ss.ROW_OK]
    assert torch.all(out[rows: 2 * rows] == 0) and torch.all(lse[rows: 2 * rows] == -math.inf)
    c.table = good
    out[rows: 2 * rows], lse[rows: 2 * rows] = run(engine, c)[0][rows: 2 * rows], run(engine, c)[1][rows: 2 * rows]
    plain.check_attend(c, out, lse, 0.125)


@pytest.mark.parametrize("rows", [1, 140])
def test_bad_rows_and_lengths_refuse_the_sequence(engine, rows):
    torch = torch_mod()
    c = plain.Case([300, 200, 250, 310], [rows] * 4, 4, 2, 64, torch.bfloat16)
    c.length[0] = -1
    c.length[1] = c.table.shape[1] * 16 + 1
    out, lse, status = run(engine, c)
    assert status.tolist() == [ss.ROW_INVALID_ROW, ss.ROW_INVALID_ROW, ss.ROW_OK, ss.ROW_OK]
    assert torch.all(out[: 2 * rows] == 0) and torch.all(out[2 * rows:].float().abs().sum(-1) > 0)
    c = plain.Case([300, 200, 250, 310], [rows] * 4, 4, 2, 64, torch.bfloat16)
    out, lse, status = run(engine, c, max_length=260)
    assert status.tolist() == [ss.ROW_INVALID_ROW, ss.ROW_OK, ss.ROW_OK, ss.ROW_INVALID_ROW]
    # starts that fall, or leave the rows: those sequences' rows are left as they were
    c.row_start = torch.tensor([0, rows, rows - 1, 3 * rows, 4 * rows + 1], dtype=torch.int32, device="cuda")
    out, lse, status = run(engine, c)
    assert status.tolist() == [ss.ROW_OK, ss.ROW_INVALID_ROW, ss.ROW_INVALID_ROW, ss.ROW_INVALID_ROW]
    assert torch.all(out[rows:] == 7.0) and torch.all(lse[rows:] == 7.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_strided_and_unaligned_rows(engine, dtype, shift):
    """q as columns of a projection's rows, out with a row stride of its own, both at odd offsets."""
    torch = torch_mod()
    for rows in ([1, 1, 1], [3, 150, 20]):
        c = plain.Case([70, 300, 41], rows, 4, 2, 64, dtype_of(dtype))
        wide = torch.randn(c.total, 4 * 64 + 37, device="cuda").to(c.dtype)
        q = wide[:, shift: shift + 256].view(c.total, 4, 64)
        q.copy_(c.q)
        room = torch.full((c.total, 300), 7.0, dtype=c.dtype, device="cuda")
        out = room[:, shift: shift + 256].view(c.total, 4, 64)
        engine.attend(q, c.cache(), c.length, 0.125, row_start=c.row_start, max_rows=c.max_rows, out=out)
        torch.cuda.synchronize()
        plain.check_attend(c, out, None, 0.125)
        assert torch.all(room[:, :shift] == 7.0) and torch.all(room[:, shift + 256:] == 7.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 100])
def test_unaligned_cache(engine, dtype, rows):
    """A pool that starts between 16-byte boundaries, with gaps between its heads."""
    torch = torch_mod()
    c = plain.Case([90, 200], [rows, rows], 4, 2, 64, dtype_of(dtype), page=32)
    pages = len(c.k)
    room = torch.full((2, pages * 32 * 2 * 67 + 1), float("nan"), dtype=c.dtype, device="cuda")
    k, v = (room[i, 1:].view(pages, 32, 2, 67)[..., :64] for i in range(2))
    k.copy_(c.k), v.copy_(c.v)
    c.k, c.v = k, v
    out, lse, _ = run(engine, c)
    plain.check_attend(c, out, lse, 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 130])
def test_offsets_past_32_bits(engine, dtype, rows):
    """A pool of more than 2^32 bytes and 2^31 elements whose last pages are the ones in use."""
    torch = torch_mod()
    c = plain.Case([300], [rows], 4, 2, 128, dtype_of(dtype), page=256, seed=5)
    pages = 2 ** 31 // (256 * 2 * 128) + 8
    room = torch.empty(2, pages, 256, 2, 128, dtype=c.dtype, device="cuda")
    for s in range(c.table.shape[1]):
        old, new = int(c.table[0, s]), pages - 1 - s
        room[0, new], room[1, new] = c.k[old], c.v[old]
        c.table[0, s] = new
    c.k, c.v = room[0], room[1]
    out, lse, _ = run(engine, c)
    plain.check_attend(c, out, lse, 128 ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 5.0])
def test_scales(engine, dtype, scale):
    c = plain.Case([150, 20], [1, 1], 4, 2, 64, dtype_of(dtype))
    out, lse, _ = run(engine, c, scale=scale)
    plain.check_attend(c, out, lse, scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 5, 300])
def test_equal_calls_give_equal_bits_on_any_stream(engine, dtype, rows):
    torch = torch_mod()
    c = plain.Case([5000, 301, 2000], [rows] * 3, 4, 2, 128, dtype_of(dtype))
    first, lse, _ = run(engine, c)
    outs = [torch.empty_like(first) for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    rooms = [engine.attend_workspace() for _ in range(4)]
    cache = c.cache()
    torch.cuda.synchronize()
    for _ in range(5):
        for o, st, room in zip(outs, streams, rooms):  # several calls of one context in flight at once
            engine.attend(c.q, cache, c.length, 128 ** -0.5, row_start=c.row_start, max_rows=rows, out=o, stream=st, workspace=room)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o.view(torch.uint8), first.view(torch.uint8))


@pytest.mark.parametrize("rows", [1, 3, 9, 30, 60])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_streams_of_all_lengths(engine, rows, dim):
    """Shares that begin and end anywhere: many sequences, idle ones among them, some longer than a share."""
    torch = torch_mod()
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, 200, (333,), generator=g).tolist()
    lens[7], lens[40], lens[41], lens[332] = 4000, 0, 0, 0
    c = plain.Case(lens, [min(rows, n) if n % 3 else rows for n in lens], 2, 1, dim, torch.bfloat16, seed=rows, fill=float("nan"))
    out, lse, status = run(engine, c, extra_rows=1)
    assert status.tolist() == [ss.ROW_OK] * 333
    plain.check_attend(c, out, lse, dim ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_length", [1, 31, 64, 96, 192, 193, 384, 385])
def test_short_bounds(engine, dtype, max_length):
    """Bounds around which a call's shares are of whole sequences and heads: lengths up to each, and one past it."""
    torch = torch_mod()
    g = torch.Generator().manual_seed(max_length)
    lens = torch.randint(0, max_length + 1, (200,), generator=g).tolist()
    lens[3], lens[150], lens[199] = max_length, 0, max_length + 1
    rows = [0 if i % 11 == 5 else 1 + i % 2 for i in range(200)]
    c = plain.Case(lens, rows, 4, 2, 64, dtype_of(dtype), seed=max_length, fill=float("nan"))
    out, lse, status = run(engine, c, max_length=max_length)
    assert status.tolist() == [ss.ROW_OK] * 199 + [ss.ROW_INVALID_ROW]
    last = c.total - rows[199]
    assert torch.all(out[last:] == 0) and torch.all(lse[last:] == -math.inf)
    want, want_lse, tol, lse_tol = plain.attend(c, 0.125)
    assert torch.all((out.double() - want).abs()[:last] <= tol[:last])
    seen = torch.isfinite(want_lse[:last])
    assert torch.equal(lse[:last][~seen].double(), want_lse[:last][~seen])
    assert torch.all((lse[:last].double() - want_lse[:last]).abs()[seen] <= lse_tol[:last][seen])


def test_more_blocks_of_rows_than_the_gpu_holds_at_once(engine):
    """Prompts whose blocks follow one another on the SMs, for many steps each."""
    torch = torch_mod()
    lens = [1100, 700, 3, 901, 256, 1300]
    c = plain.Case(lens, lens, 32, 8, 128, torch.bfloat16, page=64, seed=3, fill=float("nan"))
    out, lse, status = run(engine, c)
    assert status.tolist() == [ss.ROW_OK] * 6
    plain.check_attend(c, out, lse, 128 ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [4, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [0, 300])
def test_drafts_on_many_query_heads(engine, dtype, rows, dim, window):
    """32 to 136 pairs of a row and a query head on one key head: the largest of a step, the smallest of a prompt."""
    c = plain.Case([rows, 2500, 900 + rows, 0], [rows, rows, 1, rows], 8, 1, dim, dtype_of(dtype), page=32, seed=rows, fill=float("nan"))
    out, lse, status = run(engine, c, window=window, sinks=3, extra_rows=1)
    assert status.tolist() == [ss.ROW_OK] * 4
    plain.check_attend(c, out, lse, dim ** -0.5, window, 3)


def test_a_workspace_must_be_large_enough(engine):
    torch = torch_mod()
    c = plain.Case([400], [1], 4, 2, 128, torch.bfloat16)
    with pytest.raises(ss.SsbError) as e:
        engine.attend(c.q, c.cache(), c.length, 1.0, workspace=engine.attend_workspace()[:-16])
    assert e.value.status == ss.OUT_OF_RANGE


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 4, 40, 150])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2 ** 31 - 1, 0), (50, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_largest_windows_and_sinks(engine, dtype, rows, window, sinks):
    c = plain.Case([rows + 700, rows], [rows, rows], 8, 4, 128, dtype_of(dtype), seed=rows)
    out, lse, status = run(engine, c, window=window, sinks=sinks)
    assert status.tolist() == [ss.ROW_OK] * 2
    plain.check_attend(c, out, lse, 128 ** -0.5, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 6, 130])
@pytest.mark.parametrize("dim", [64, 80])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 170, 60])
def test_windows_longer_than_sequences_with_idle_rows(engine, dtype, rows, dim, window):
    """Rows before position 0 leave those after them what they see, however far back the window reaches."""
    lens = [1, rows - 1, rows // 2, 40 + rows, 0]
    c = plain.Case(lens, [rows] * 5, 4, 2, dim, dtype_of(dtype), seed=rows, fill=float("nan"))
    out, lse, status = run(engine, c, ragged=False, window=window, sinks=2)
    assert status.tolist() == [ss.ROW_OK] * 5
    plain.check_attend(c, out, lse, dim ** -0.5, window, 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 20, 150])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("at", [5, 61, "last"])
def test_infinities_that_are_seen(engine, dtype, rows, dim, at):
    """A key that scores -inf has a weight of 0, as one far below the others; a value's infinity reaches its own element only."""
    torch = torch_mod()
    c = plain.Case([200 + rows], [rows], 4, 2, dim, dtype_of(dtype), seed=rows)
    c.q[..., 0] = c.q[..., 0].abs() + 0.5
    at = 200 if at == "last" else at  # the position of the first row: the last that all of them see
    page, slot = int(c.table[0, at // c.page]), at % c.page
    kept = c.k[page, slot].clone(), c.v[page, slot].clone()
    c.k[page, slot, :, 0] = -2.0 ** 15  # a score below -1500: its weight rounds to 0
    want = run(engine, c)
    c.k[page, slot, :, 0] = float("-inf")
    got = run(engine, c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    c.k[page, slot] = kept[0]
    c.v[page, slot, :, 3] = float("inf")
    out, lse, _ = run(engine, c)
    assert torch.all(out[..., 3] == float("inf"))
    c.v[page, slot] = kept[1]
    out[..., 3] = run(engine, c)[0][..., 3]
    plain.check_attend(c, out, lse, dim ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 5, 90, 300])
@pytest.mark.parametrize("dim", [64, 80, 128])
def test_in_place(engine, dtype, rows, dim):
    """out may be q: a pair's query is read before anything of its output is written."""
    torch = torch_mod()
    c = plain.Case([rows + 4000, rows], [rows, rows], 4, 2, dim, dtype_of(dtype), seed=rows)
    want, lse, _ = run(engine, c)
    q = c.q.clone()
    engine.attend(q, c.cache(), c.length, dim ** -0.5, row_start=c.row_start, max_rows=rows, out=q)
    torch.cuda.synchronize()
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("max_rows", [1, 200])
def test_calls_without_rows(engine, max_rows):
    """No sequence, or only sequences without a row: the statuses are all that is written."""
    torch = torch_mod()
    c = plain.Case([40, 30], [1, 1], 4, 2, 64, torch.bfloat16)
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    status = torch.full((2,), -7, dtype=torch.int32, device="cuda")
    q = c.q[:0]
    for _ in range(2):
        engine.attend(q, c.cache(), c.length, 0.125, row_start=none, max_rows=max_rows, status=status)
        engine.norm_rope_append(q, q[:, :2], q[:, :2], c.cache(), c.length, None, row_start=none, max_rows=max_rows, status=status)
    torch.cuda.synchronize()
    assert status.tolist() == [ss.ROW_OK] * 2
    out = torch.full_like(c.q, 7.0)  # rows that belong to no sequence
    engine.attend(c.q, c.cache(), c.length, 0.125, row_start=none, max_rows=max_rows, out=out)
    empty = ss.KvCache(c.k, c.v, torch.zeros(0, 4, dtype=torch.int32, device="cuda"))
    engine.attend(c.q, empty, c.length[:0], 0.125, max_rows=max_rows, out=out)
    torch.cuda.synchronize()
    assert torch.all(out == 7.0)


@pytest.mark.parametrize("rows", [1, 3, 200])
def test_a_captured_call_follows_the_device_lengths(engine, rows):
    torch = torch_mod()
    c = plain.Case([rows + 400, rows + 300], [rows, rows], 4, 2, 128, torch.bfloat16)
    cache, out, lse = c.cache(), torch.empty_like(c.q), torch.empty(2 * rows, 4, device="cuda")

    def call():
        engine.attend(c.q, cache, c.length, 128 ** -0.5, max_rows=rows, out=out, lse=lse, stream=torch.cuda.current_stream())

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([rows + 400, rows + 300], [1, 300], [0, 17], [rows + 399, 64]):
        c.lens = lens
        c.length.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        plain.check_attend(c, out, lse, 128 ** -0.5)


@pytest.mark.parametrize("rows", [1, 200])
def test_two_graphs_with_workspaces_of_their_own_run_at_once(engine, rows):
    torch = torch_mod()
    cases = [plain.Case([9000, 41 + rows], [rows, rows], 4, 2, 128, torch.bfloat16, seed=s) for s in (1, 2)]
    outs, graphs, rooms = [], [], []
    for c in cases:
        out, room, cache = torch.empty_like(c.q), engine.attend_workspace(), c.cache()

        def call(c=c, out=out, room=room, cache=cache):
            engine.attend(c.q, cache, c.length, 128 ** -0.5, max_rows=rows, out=out, stream=torch.cuda.current_stream(), workspace=room)

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(8):
                call()
        outs.append(out), graphs.append(graph), rooms.append((room, cache))
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for c, out in zip(cases, outs):
        plain.check_attend(c, out, None, 128 ** -0.5)


@pytest.mark.parametrize("pairs", [(3, 1), (5, 1), (4, 5), (4, 16), (8, 20)])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("value", ["max", "min"])
@pytest.mark.parametrize("seen_by", ["all", "last"])
def test_largest_values(engine, pairs, dim, value, seen_by):
    """The largest fp32 numbers as values: what sees them takes them as they are, what does not see them nothing."""
    torch = torch_mod()
    group, rows = pairs
    c = plain.Case([700 + rows, 40], [rows, 1], group, 1, dim, torch.float32, seed=rows)
    large = getattr(torch.finfo(torch.float32), value)
    at = 700 if seen_by == "all" else c.lens[0] - 1
    page, slot = c.table[0, at // c.page].long(), at % c.page
    c.v[page, slot, :, 1] = large
    c.v[page, slot, :, dim - 2] = -large
    c.v[page, slot, :, 5] = torch.tensor(0x7f7ff000, dtype=torch.int32).view(torch.float32).item()  # rounds up to 2^128 in 11 bits
    c.v[page, slot, :, 6] = torch.tensor(0x7f7fefff, dtype=torch.int32).view(torch.float32).item()  # and this one does not
    out, lse, _ = run(engine, c)
    assert torch.isfinite(out).all()
    plain.check_attend(c, out, lse, dim ** -0.5)


@pytest.mark.parametrize("seqs,rows", [(1, 150), (1, 300), (20, 150)])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("growth", [0.0, 7.5, 40.0])
def test_largest_bf16_values(engine, rows, seqs, dim, growth):
    """A value of the largest size behind steps of smaller scores: no partial output is larger than what it is a part of. The
    scores are 0 but for one position's, `growth` in units of the base 2 logarithm."""
    torch = torch_mod()
    c = plain.Case([rows + 300] * seqs, [rows] * seqs, 4, 2, dim, torch.bfloat16, page=64, seed=rows)
    c.q.zero_(), c.k.zero_()
    c.q[..., 0] = 1.0
    at = 290  # seen by all rows, behind two steps of 128 positions
    largest = torch.finfo(torch.bfloat16).max
    for s in range(seqs):
        page, slot = c.table[s, at // c.page].long(), at % c.page
        c.k[page, slot, :, 0] = growth
        c.v[page, slot, :, 1], c.v[page, slot, :, dim - 1] = largest, -largest
    out, lse, _ = run(engine, c, scale=math.log(2.0))
    assert torch.isfinite(out).all()
    plain.check_attend(c, out, lse, math.log(2.0))


@pytest.mark.parametrize("captured", [False, True])
def test_contexts_allocate_their_workspace_with_their_first_call(engine, captured):
    """A context that only samples holds none, and a context's first call may be one that a graph captures."""
    torch = torch_mod()
    c = plain.Case([3000, 41], [1, 1], 4, 2, 128, torch.bfloat16)
    want, want_lse, _ = run(engine, c)
    cache, out, lse = c.cache(), torch.empty_like(c.q), torch.empty(2, 4, device="cuda")
    fresh = [ss.Sampler(0) for _ in range(1 if captured else 8)]
    size = engine.attend_workspace().numel()

    def call(e):
        e.attend(c.q, cache, c.length, 128 ** -0.5, row_start=c.row_start, out=out, lse=lse, stream=torch.cuda.current_stream())

    try:
        torch.cuda.synchronize()
        free = torch.cuda.mem_get_info()[0]
        for e in fresh:
            if captured:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    call(e)
            for _ in range(2):
                out.fill_(7.0), lse.fill_(7.0)
                graph.replay() if captured else call(e)
                torch.cuda.synchronize()
                assert torch.equal(out, want) and torch.equal(lse, want_lse)
        if not captured:  # (memory that the driver still holds from before is taken first)
            assert free - torch.cuda.mem_get_info()[0] >= 4 * size
    finally:
        for e in fresh:
            e.close()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 6, 140])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-40, -1e-38])
def test_scales_next_to_zero(engine, dtype, rows, scale):
    """Scores of any size times a scale of 0 weigh the same; an infinite one is not a number then, and -inf for a scale above 0."""
    torch = torch_mod()
    c = plain.Case([260 + rows, rows], [rows, rows], 4, 2, 64, dtype_of(dtype), seed=rows)
    c.q.mul_(1e17), c.k.mul_(1e17)
    out, lse, _ = run(engine, c, scale=scale)
    plain.check_attend(c, out, lse, scale)
    c.q.abs_().mul_(1e-17), c.k.mul_(1e-17)
    page, slot = c.table[0, 200 // c.page].long(), 200 % c.page
    c.k[page, slot] = float("-inf") if scale >= 0 else float("inf")  # a score of -inf, where the scale is not 0
    out, lse, _ = run(engine, c, scale=scale)
    if scale == 0.0:
        assert torch.isnan(out[:rows]).all() and torch.isnan(lse[:rows]).all()
    else:
        c.k[page, slot] = 0.0  # the position's weight is 0 and the others' are 1, to 2^-24
        assert torch.isfinite(out).all()
        v = c.gathered(0)[1]
        for i in range(rows):
            seen = [j for j in range(261 + i) if j != 200]
            want = v[seen].mean(0).repeat_interleave(2, 0)
            bound = (2 * (72 + len(seen)) * plain.U + 2.0 ** -8 * (dtype == "bf16")) * v[seen].abs().mean(0).repeat_interleave(2, 0)
            assert torch.all((out[i].double() - want).abs() <= bound + 2.0 ** -8 * (dtype == "bf16") * want.abs())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 5, 40, 200])
@pytest.mark.parametrize("max_length", [330, 4000])
def test_statuses_of_replayed_calls(engine, dtype, rows, max_length):
    """Each replay of a captured call clears the statuses that the one before has raised."""
    torch = torch_mod()
    c = plain.Case([300 + rows, 250, 4000], [rows] * 3, 4, 2, 128, dtype_of(dtype))
    cache, out = c.cache(), torch.empty_like(c.q)
    status = torch.full((3,), -7, dtype=torch.int32, device="cuda")
    good, page = c.length.clone(), int(c.table[1, 2])

    def call():
        engine.attend(c.q, cache, c.length, 128 ** -0.5, row_start=c.row_start, max_rows=rows, max_length=max_length, out=out, status=status,
                      stream=torch.cuda.current_stream())

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    long = [ss.ROW_INVALID_ROW if n > max_length else ss.ROW_OK for n in c.lens]
    for length, entry, want in ((None, page, long), (-1, page, [long[0], ss.ROW_INVALID_ROW, long[2]]), (None, page, long),
                                (None, -1, [long[0], ss.ROW_INVALID_ROW, long[2]]), (0, page, long), (None, page, long)):
        c.length.copy_(good)
        if length is not None:
            c.length[1] = length
        c.table[1, 2] = entry
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert status.tolist() == want
