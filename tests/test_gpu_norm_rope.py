"""Head norms, rotation and cache append in one pass (ssb_norm_rope_append) against the plain form in 64 bits;
the tolerances are derived in decoder_plain.py."""
import pytest

import decoder_plain as plain
import speech_sampler as ss

pytestmark = pytest.mark.gpu


def torch_mod():
    import torch
    return torch


def dtype_of(name):
    torch = torch_mod()
    return torch.float32 if name == "f32" else torch.bfloat16


def freqs(rope):
    torch = torch_mod()
    half = rope // 2
    return 1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(half, 1))


def close(got, want, err):
    torch = torch_mod()
    half = torch.finfo(got.dtype).eps / 2
    off = (got.double() - want).abs()
    return bool(torch.all(off <= err + half * (want.abs() + err)))


def rows_of(c):
    """(sequence, position) of each row."""
    out = []
    for s, (n, r) in enumerate(zip(c.lens, c.rows)):
        out.extend((s, n - r + i) for i in range(r))
    return out


def call_and_check(engine, c, rope=None, interleaved=False, dtype=None, q_weight=True, k_weight=True, positions=None,
                   in_place=False, extra_rows=0, ragged=True, eps=1e-6, shift=0, refused=()):
    torch = torch_mod()
    rope = c.dim if rope is None else rope
    dtype = c.dtype if dtype is None else dtype
    n, width = c.total + extra_rows, (c.heads + 2 * c.kv_heads) * c.dim
    room = torch.randn(n, width + 9, device="cuda", generator=c.gen).to(dtype)
    qkv = room[:, shift: shift + width]
    a, b = c.heads * c.dim, (c.heads + c.kv_heads) * c.dim
    q, k, v = (x.view(n, -1, c.dim) for x in (qkv[:, :a], qkv[:, a:b], qkv[:, b:]))
    qw = 1 + 0.4 * torch.randn(c.dim, device="cuda", generator=c.gen) if q_weight else None
    kw = 1 + 0.4 * torch.randn(c.dim, device="cuda", generator=c.gen) if k_weight else None
    f = freqs(rope)
    before_k, before_v, q0, k0, v0 = c.k.clone(), c.v.clone(), q.clone(), k.clone(), v.clone()
    status = torch.full((len(c.lens),), -7, dtype=torch.int32, device="cuda")
    q_out = q if in_place else torch.full((n, c.heads, c.dim), 7.0, dtype=dtype, device="cuda")
    engine.norm_rope_append(q, k, v, c.cache(), c.length, f, qw, kw, eps, interleaved, c.row_start if ragged else None,
                            c.max_rows, positions, q_out, status)
    torch.cuda.synchronize()
    where = rows_of(c)
    assert torch.equal(q_out[c.total:], q0[c.total:] if in_place else torch.full_like(q_out[c.total:], 7.0))
    assert torch.equal(k, k0) and torch.equal(v, v0)
    live = [i for i, (s, p) in enumerate(where) if p >= 0 and s not in refused]
    idle = [i for i in range(c.total) if i not in live]
    assert torch.all(q_out[idle] == 0)
    at = torch.tensor([p for _, p in where], device="cuda") if positions is None else positions[: c.total]
    want, err = plain.norm_rope(q0[: c.total], qw, eps, at, f, interleaved)
    assert close(q_out[live], want[live], err[live])
    want, err = plain.norm_rope(k0[: c.total], kw, eps, at, f, interleaved)
    if live:
        page = torch.tensor([int(c.table[where[i][0], where[i][1] // c.page]) for i in live], device="cuda")
        slot = torch.tensor([where[i][1] % c.page for i in live], device="cuda")
        assert close(c.k[page, slot], want[live], err[live])
        assert torch.equal(c.v[page, slot], v0[live].to(c.v.dtype))
        before_k[page, slot], before_v[page, slot] = c.k[page, slot], c.v[page, slot]
    assert torch.equal(c.k, before_k) and torch.equal(c.v, before_v)  # nothing else is written
    return status.tolist()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,rows", [([1], [1]), ([17, 64, 65], [1, 1, 1]), ([9, 100], [9, 33]), ([40, 0, 7, 300], [3, 0, 7, 250])])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rows(engine, dtype, lens, rows, interleaved):
    c = plain.Case(lens, rows, 4, 2, 128, dtype_of(dtype), seed=sum(lens))
    assert call_and_check(engine, c, interleaved=interleaved, extra_rows=2) == [ss.ROW_OK] * len(lens)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (7, 1), (32, 8), (40, 2)])
@pytest.mark.parametrize("dim,rope", [(16, 16), (64, 32), (80, 80), (80, 40), (128, 64), (128, 8), (128, 0), (256, 256), (256, 96)])
def test_head_layouts(engine, heads, kv_heads, dim, rope):
    for interleaved in (False, True):
        c = plain.Case([33, 130], [1, 5], heads, kv_heads, dim, dtype_of("bf16"), 32, "positions", seed=dim + heads)
        call_and_check(engine, c, rope, interleaved)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cache_dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 256])
def test_types_and_pages(engine, dtype, cache_dtype, page):
    c = plain.Case([70, 257], [5, 30], 4, 2, 64, dtype_of(cache_dtype), page)
    call_and_check(engine, c, dtype=dtype_of(dtype))


@pytest.mark.parametrize("q_weight", [False, True])
@pytest.mark.parametrize("k_weight", [False, True])
def test_without_norms(engine, q_weight, k_weight):
    c = plain.Case([70, 20], [5, 1], 4, 2, 64, dtype_of("f32"))
    call_and_check(engine, c, q_weight=q_weight, k_weight=k_weight)


def test_far_positions(engine):
    """Angles of positions up to 2^31 - 1, and negative ones: the product with the frequency is reduced in 64 bits."""
    torch = torch_mod()
    c = plain.Case([300], [8], 2, 1, 128, torch.float32)
    far = torch.tensor([0, 1, 10 ** 5, 10 ** 6, 2 ** 24 + 1, 2 ** 31 - 1, -5, -2 ** 31], dtype=torch.int32, device="cuda")
    call_and_check(engine, c, positions=far)


@pytest.mark.parametrize("shift", [0, 1, 2])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place_and_unaligned(engine, shift, dtype):
    c = plain.Case([70, 20, 500], [5, 1, 450], 4, 2, 64, dtype_of(dtype))
    call_and_check(engine, c, in_place=True, shift=shift, extra_rows=1)
    call_and_check(engine, c, shift=shift)


def test_many_rows_and_streams(engine):
    """More streams than a warp finds in one step, and rows enough for one CTA each."""
    torch = torch_mod()
    g = torch.Generator().manual_seed(1)
    rows = torch.randint(0, 4, (1300,), generator=g).tolist()
    rows[0] = rows[-1] = 0
    lens = [r + int(torch.randint(0, 40, (1,), generator=g)) for r in rows]
    c = plain.Case(lens, rows, 2, 1, 16, torch.bfloat16)
    assert call_and_check(engine, c) == [ss.ROW_OK] * 1300


def test_idle_and_refused_sequences(engine):
    torch = torch_mod()
    c = plain.Case([0, 40, 2, 60], [3, 3, 3, 3], 4, 2, 64, torch.float32)
    assert call_and_check(engine, c, ragged=False) == [ss.ROW_OK] * 4
    c.length[1] = -4
    c.length[3] = c.table.shape[1] * 16 + 1
    assert call_and_check(engine, c, ragged=False, refused=(1, 3)) == [ss.ROW_OK, ss.ROW_INVALID_ROW, ss.ROW_OK, ss.ROW_INVALID_ROW]


@pytest.mark.parametrize("page_id", [-1, -2 ** 31, 2 ** 31 - 1])
def test_a_bad_page_skips_its_rows(engine, page_id):
    torch = torch_mod()
    c = plain.Case([40, 40], [1, 1], 4, 2, 64, torch.bfloat16)
    c.table[1, 2] = page_id
    assert call_and_check(engine, c, refused=(1,)) == [ss.ROW_OK, ss.ROW_INVALID_ROW]
    c.table[1, 0] = page_id  # a page behind the new row is not looked at
    c.table[1, 2] = int(c.table[0, 0])
    assert call_and_check(engine, c) == [ss.ROW_OK, ss.ROW_OK]


def test_offsets_past_32_bits(engine):
    torch = torch_mod()
    c = plain.Case([300], [60], 4, 2, 128, torch.bfloat16, page=256, seed=5)
    pages = 2 ** 31 // (256 * 2 * 128) + 8
    k, v = torch.zeros(2, pages, 256, 2, 128, dtype=torch.bfloat16, device="cuda")
    c.table[0] = torch.tensor([pages - 1, pages - 2], dtype=torch.int32)
    c.k, c.v = k, v
    call_and_check(engine, c)


def test_a_captured_call_appends_where_the_lengths_say(engine):
    torch = torch_mod()
    c = plain.Case([100, 90], [1, 1], 4, 2, 64, torch.bfloat16)
    q, k, v = (torch.randn(2, h, 64, device="cuda").to(torch.bfloat16) for h in (4, 2, 2))
    f, cache, out = freqs(64), c.cache(), torch.empty_like(q)

    def call():
        engine.norm_rope_append(q, k, v, cache, c.length, f, q_out=out, stream=torch.cuda.current_stream())

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([100, 90], [1, 64], [17, 0]):
        c.length.copy_(torch.tensor(lens, dtype=torch.int32))
        c.v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for s, n in enumerate(lens):
            if n:
                p = n - 1
                assert torch.equal(c.v[int(c.table[s, p // 16]), p % 16], v[s])
        assert int((c.v != 0).any(-1).any(-1).sum()) == sum(n > 0 for n in lens)


@pytest.mark.parametrize("seqs", [4, 75])
@pytest.mark.parametrize("bad", [1, 2])
def test_a_falling_start_refuses_its_own_sequences_only(engine, seqs, bad):
    """One start too low: the sequence that ends there has less than no rows, the one that begins there too many; the rows
    of the others, on both sides, are appended. A row that two sequences claim is the one's that may have it."""
    torch = torch_mod()
    rows = 6
    c = plain.Case([50 + s for s in range(seqs)], [rows] * seqs, 4, 2, 64, torch.bfloat16, seed=seqs)
    starts = [rows * s for s in range(seqs + 1)]
    starts[bad + 1] = starts[bad] - 1
    row_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    n = c.total
    q, k, v = (torch.randn(n, h, 64, device="cuda", generator=c.gen).to(c.dtype) for h in (4, 2, 2))
    out = torch.full_like(q, 7.0)
    status = torch.full((seqs,), -7, dtype=torch.int32, device="cuda")
    before_k, before_v, f = c.k.clone(), c.v.clone(), freqs(64)
    engine.norm_rope_append(q, k, v, c.cache(), c.length, f, row_start=row_start, max_rows=rows, q_out=out, status=status)
    torch.cuda.synchronize()
    refused = (bad, bad + 1)
    assert status.tolist() == [ss.ROW_INVALID_ROW if s in refused else ss.ROW_OK for s in range(seqs)]
    where = [(s, c.lens[s] - rows + i) for s in range(seqs) for i in range(rows)]
    live = torch.tensor([i for i, (s, _) in enumerate(where) if s not in refused], device="cuda")
    at = torch.tensor([p for _, p in where], device="cuda")
    want, err = plain.norm_rope(q, None, 1e-6, at, f, False)
    assert close(out[live], want[live], err[live])
    assert torch.all(out[bad * rows: (bad + 2) * rows] == 7.0)  # left as they were
    page = torch.tensor([int(c.table[where[i][0], where[i][1] // c.page]) for i in live.tolist()], device="cuda")
    slot = at[live] % c.page
    want, err = plain.norm_rope(k, None, 1e-6, at, f, False)
    assert close(c.k[page, slot], want[live], err[live]) and torch.equal(c.v[page, slot], v[live])
    before_k[page, slot], before_v[page, slot] = c.k[page, slot], c.v[page, slot]
    assert torch.equal(c.k, before_k) and torch.equal(c.v, before_v)  # nothing else is written
