"""Failure detection of the decoder step without a GPU fault: the attention kernels' bounded waits.

The wait-limit test library (the engine's sources built with SSB_WAIT_TEST: waits give up after about 2 ms) never issues the
copies of the third tile of sequence 1's second key head, nor, in a prompt, those of the third step of that head's last
block of rows, where there are several. Everything that waits for them gives up, in a step's share also what comes after them.
What was given up is NaN and its sequence SSB_ROW_DEVICE_TIMEOUT, everything else is right, no kernel faults or hangs, and
afterwards both the same library (on sequences that do not reach the gap) and the product library serve normal calls."""
import os

import pytest

import decoder_plain as plain
import speech_sampler as ss

pytestmark = pytest.mark.gpu
WAITTEST = os.path.join(os.path.dirname(ss.LIB_PATH), "libspeech_sampler_b200_waittest.so")


@pytest.fixture(scope="module")
def gap(engine):
    """An engine of the wait-limit test library (and the product's, loaded before)."""
    assert os.path.exists(WAITTEST), "the wait-limit test library is not built (speech_build.py builds it)"
    product, ss._LIB = ss._LIB, None
    try:
        ss.load_library(WAITTEST)
        s = ss.Sampler(0)
    finally:
        ss._LIB = product
    yield s
    s.close()


def call(engine, c, max_length=0):
    import torch
    out = torch.full((c.total, c.heads, c.dim), 7.0, dtype=c.dtype, device="cuda")
    lse = torch.full((c.total, c.heads), 7.0, device="cuda")
    status = torch.full((len(c.lens),), -7, dtype=torch.int32, device="cuda")
    engine.attend(c.q, c.cache(), c.length, c.dim ** -0.5, row_start=c.row_start, max_rows=c.max_rows, max_length=max_length, out=out,
                  lse=lse, status=status)
    torch.cuda.synchronize()  # raises if the kernel faulted
    return out, lse, status


def given_up(c, out):
    """[rows, heads]: whether a row and head is NaN; the others have to be right."""
    import torch
    want, _, tol, _ = plain.attend(c, c.dim ** -0.5)
    nan = torch.isnan(out).all(-1)
    assert torch.all(((out.double() - want).abs() <= tol).all(-1) | nan)
    return nan


def check_statuses(c, nan, status):
    """A sequence of which something was given up says so, whoever of its heads and blocks came last, and no other does."""
    want = [ss.ROW_DEVICE_TIMEOUT if nan[rows_of(c, s)].any() else ss.ROW_OK for s in range(len(c.lens))]
    assert status.tolist() == want and want[1] == ss.ROW_DEVICE_TIMEOUT


def rows_of(c, s):
    return slice(int(c.row_start[s]), int(c.row_start[s + 1]))


def normal_calls(engine, gap, c):
    """Sequences of fewer than three tiles on the library with the gap, and the same call on the product's."""
    short = plain.Case([50, 60, 33], [1, 2, 1], c.heads, c.kv_heads, c.dim, c.dtype)
    for s, case in ((gap, short), (engine, short), (engine, c)):
        out, lse, status = call(s, case)
        assert status.tolist() == [ss.ROW_OK] * len(case.lens)
        plain.check_attend(case, out, lse, case.dim ** -0.5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,rows", [(2, 1), (4, 2), (8, 5), (8, 10)])
@pytest.mark.parametrize("longest", [190, 3000])
def test_a_step_gives_up(engine, gap, dtype, dim, heads, rows, longest):
    """Shares of whole units (up to 192 positions) and cut ones; 1 to 40 pairs of a key head."""
    import torch
    lens = [longest, longest - 10, 70, longest - 3, 0, longest // 2, 190, 1]
    c = plain.Case(lens, [min(rows, max(n, 1)) for n in lens], heads, 2, dim, torch.float32 if dtype == "f32" else torch.bfloat16)
    half = heads // 2
    for _ in range(2):
        out, lse, status = call(gap, c, max_length=longest)
        nan = given_up(c, out)
        check_statuses(c, nan, status)
        assert nan[rows_of(c, 1), half:].all()
        if longest <= 192:  # a unit per share: nothing else is lost
            nan[rows_of(c, 1), half:] = False
            assert not nan.any()
    normal_calls(engine, gap, c)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("longest", [300, 900])
def test_a_prompt_gives_up(engine, gap, dim, longest):
    """Blocks of 256 pairs in CTAs of their own (20 sequences fill the GPU); the third step is the last one issued, or not."""
    import torch
    lens = [longest, longest - 1] + [longest - 20 * i for i in range(14)] + [0, 1, 250, 17]
    c = plain.Case(lens, [min(n, 200) for n in lens], 8, 4, dim, torch.bfloat16)
    for _ in range(2):
        out, lse, status = call(gap, c, max_length=longest)
        nan = given_up(c, out)
        check_statuses(c, nan, status)
        first = int(c.row_start[1])
        assert nan[first + 128: first + 200, 2:4].all()  # pairs 256 and on of key head 1
        nan[first + 128: first + 200, 2:4] = False
        assert not nan.any()
    normal_calls(engine, gap, c)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_timeout_next_to_a_joined_head(engine, gap, dtype):
    """Sequences of 4 tiles in shares of 5 places, each unit 2 places and its tiles: sequence 1's first head is cut by a share and
    joined after the second, which is whole, gave up."""
    import torch
    tile = 32 if dtype == "f32" else 64
    c = plain.Case([4 * tile] * 100 + [8 * tile], [1] * 101, 2, 2, 128, torch.float32 if dtype == "f32" else torch.bfloat16)
    for _ in range(3):
        out, lse, status = call(gap, c)
        nan = given_up(c, out)
        assert nan[1, 1] and not nan[1, 0]
        check_statuses(c, nan, status)


def test_a_timeout_before_the_first_block(engine, gap):
    """Prompts whose last blocks, which start first, give up long before their first ones are done."""
    import torch
    c = plain.Case([10000] * 20, [10000] * 20, 32, 8, 128, torch.bfloat16, page=128)
    want, want_lse, want_status = call(engine, c)
    assert want_status.tolist() == [ss.ROW_OK] * 20
    out, lse, status = call(gap, c)
    nan = torch.isnan(out).all(-1)
    rows = c.rows[0]
    first = (rows * 4 - 1) // 256 * 256 // 4  # of the last block
    lost = torch.zeros_like(nan)
    lost[rows + first: 2 * rows, 4:8] = True
    assert torch.equal(nan, lost) and torch.equal(torch.isinf(lse), lost)
    assert torch.equal(out[~lost], want[~lost]) and torch.equal(lse[~lost], want_lse[~lost])
    check_statuses(c, nan, status)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("longest", [300, 700, 2100])
def test_a_prompt_shared_by_a_cluster_gives_up(engine, gap, dim, longest):
    """2, 4 and 8 CTAs share the positions of a block: where one of them gives up the block is lost, not joined as zeros."""
    import torch
    c = plain.Case([longest, longest - 1, 250], [200, 200, 200], 4, 2, dim, torch.bfloat16)
    for _ in range(2):
        out, lse, status = call(gap, c)
        nan = given_up(c, out)
        check_statuses(c, nan, status)
        assert nan[328:400, 2:4].all() and torch.all(lse[328:400, 2:4] == -float("inf"))
        nan[328:400, 2:4] = False
        assert not nan.any()
    normal_calls(engine, gap, c)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [5, 10, 16])
@pytest.mark.parametrize("tiles", [5, 6, 11])
def test_one_warp_of_a_group_gives_up(engine, gap, dtype, dim, rows, tiles):
    """The wait-limit test library lets the last warp of 16 pairs give up on a tile that the others of its group had: whether that
    group joins (5 tiles) or hands over (6), or the unit is cut (11), its pairs are not mixed with what was lost."""
    import torch
    n = tiles * (32 if dtype == "f32" else 64)
    lens = [40, 30, n - 3, 50, n]
    c = plain.Case(lens, [rows] * 5, 8, 2, dim, torch.float32 if dtype == "f32" else torch.bfloat16)
    for _ in range(2):
        out, lse, status = call(gap, c, max_length=n)
        nan = given_up(c, out)
        want = [ss.ROW_DEVICE_TIMEOUT if nan[rows_of(c, s)].any() else ss.ROW_OK for s in range(5)]
        assert status.tolist() == want
        last = torch.arange(rows * 4, device="cuda").view(rows, 4) // 16 == (rows * 4 - 1) // 16  # pairs of the last warp
        assert nan[rows_of(c, 2), 4:][last].all()
    normal_calls(engine, gap, c)
