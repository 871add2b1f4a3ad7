"""The decoder-step entry points refuse bad arguments on the host before touching a device. CPU only."""
import ctypes

import pytest

import speech_sampler as ss


@pytest.fixture(scope="module")
def lib():
    import speech_build
    speech_build.build()
    return ss.load_library()


def cache(**kw):
    c = ss.KvCacheStruct(0x1000, 0x2000, ss.BF16, 4, 16, 2, 64, 0, 2048, 64, 1024, 0x3000, 8)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def rows(**kw):
    r = ss.KvRows(2, 2, 1, 0, None, 0x4000, None)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def attend(**kw):
    a = ss.Attend(0x5000, 256, 4, ss.BF16, 0.125, 0, 0, 0, 0x6000, 256, None, None, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def norm_rope(**kw):
    n = ss.NormRope(0x5000, 0x6000, 0x7000, 256, 128, 128, 4, ss.BF16, None, None, 1e-6, 64, 0, 0, 0x8000, None, 0x9000, 256)
    for k, v in kw.items():
        setattr(n, k, v)
    return n


def test_struct_layouts():
    assert ctypes.sizeof(ss.KvCacheStruct) == 80 and ctypes.sizeof(ss.KvRows) == 40
    assert ctypes.sizeof(ss.NormRope) == 120 and ctypes.sizeof(ss.Attend) == 80
    assert bytes(rows()) == ss._PACK_ROWS.pack(2, 2, 1, 0, 0, 0x4000, 0)
    assert bytes(attend(window=7, sinks=8, max_length=9, lse=0x1, workspace=0x2, workspace_bytes=3)) == ss._PACK_ATTEND.pack(
        0x5000, 256, 4, ss.BF16, 0.125, 7, 8, 9, 0x6000, 256, 0x1, 0x2, 3)
    assert bytes(norm_rope(q_weight=0x1, k_weight=0x2, positions=0x3, interleaved=1)) == ss._PACK_NORM_ROPE.pack(
        0x5000, 0x6000, 0x7000, 256, 128, 128, 4, ss.BF16, 0x1, 0x2, 1e-6, 64, 1, 0, 0x8000, 0x3, 0x9000, 256)


BAD_CACHE = [("dtype", 2, ss.INVALID_ARGUMENT, "dtype"), ("page_size", 8, ss.INVALID_ARGUMENT, "page_size"),
             ("page_size", 24, ss.INVALID_ARGUMENT, "page_size"), ("page_size", 512, ss.INVALID_ARGUMENT, "page_size"),
             ("head_dim", 0, ss.INVALID_ARGUMENT, "head_dim"), ("head_dim", 72, ss.INVALID_ARGUMENT, "head_dim"),
             ("head_dim", 272, ss.INVALID_ARGUMENT, "head_dim"), ("kv_heads", 0, ss.INVALID_ARGUMENT, "kv_heads"),
             ("kv_heads", 2000, ss.OUT_OF_RANGE, "SSB_MAX_HEADS"), ("pages", -1, ss.INVALID_ARGUMENT, "pages"),
             ("table_ld", -1, ss.INVALID_ARGUMENT, "table_ld"), ("reserved", 1, ss.INVALID_ARGUMENT, "reserved"),
             ("page_stride", -2048, ss.INVALID_ARGUMENT, "strides"), ("position_stride", 63, ss.INVALID_ARGUMENT, "strides"),
             ("head_stride", 63, ss.INVALID_ARGUMENT, "strides"), ("table", None, ss.INVALID_ARGUMENT, "table"),
             ("k", None, ss.INVALID_ARGUMENT, "k and v"), ("v", None, ss.INVALID_ARGUMENT, "k and v")]
BAD_ROWS = [("seqs", -1, ss.INVALID_ARGUMENT, "seqs"), ("rows", -1, ss.INVALID_ARGUMENT, "rows"),
            ("seqs", 65537, ss.OUT_OF_RANGE, "SSB_MAX_SEQUENCES"), ("rows", 1048577, ss.OUT_OF_RANGE, "SSB_MAX_ROWS"),
            ("max_rows", 0, ss.INVALID_ARGUMENT, "max_rows"), ("max_rows", 1048577, ss.OUT_OF_RANGE, "SSB_MAX_ROWS"),
            ("max_rows", 2, ss.INVALID_ARGUMENT, "row_start"), ("reserved", 1, ss.INVALID_ARGUMENT, "reserved"),
            ("length", None, ss.INVALID_ARGUMENT, "length")]
BAD_ATTEND = [("dtype", ss.F32, ss.INVALID_ARGUMENT, "dtype"), ("q_heads", 0, ss.INVALID_ARGUMENT, "q_heads"),
              ("q_heads", 3, ss.INVALID_ARGUMENT, "q_heads"), ("q_heads", 1026, ss.OUT_OF_RANGE, "SSB_MAX_HEADS"),
              ("scale", float("nan"), ss.INVALID_ARGUMENT, "scale"), ("scale", float("inf"), ss.INVALID_ARGUMENT, "scale"),
              ("scale", 3e38, ss.INVALID_ARGUMENT, "scale"),
              ("window", -1, ss.INVALID_ARGUMENT, "window"), ("sinks", -1, ss.INVALID_ARGUMENT, "sinks"),
              ("max_length", -1, ss.INVALID_ARGUMENT, "max_length"), ("q_ld", 255, ss.INVALID_ARGUMENT, "q_ld"),
              ("out_ld", 255, ss.INVALID_ARGUMENT, "out_ld"), ("q", None, ss.INVALID_ARGUMENT, "q and out"),
              ("out", None, ss.INVALID_ARGUMENT, "q and out"), ("workspace", 0x1008, ss.INVALID_ARGUMENT, "workspace")]
BAD_NORM_ROPE = [("dtype", 5, ss.INVALID_ARGUMENT, "dtype"), ("q_heads", 0, ss.INVALID_ARGUMENT, "q_heads"),
                 ("q_heads", 2000, ss.OUT_OF_RANGE, "SSB_MAX_HEADS"), ("rope_dim", -8, ss.INVALID_ARGUMENT, "rope_dim"),
                 ("rope_dim", 4, ss.INVALID_ARGUMENT, "rope_dim"), ("rope_dim", 72, ss.INVALID_ARGUMENT, "rope_dim"),
                 ("interleaved", 2, ss.INVALID_ARGUMENT, "interleaved"), ("reserved", 1, ss.INVALID_ARGUMENT, "reserved"),
                 ("eps", -1.0, ss.INVALID_ARGUMENT, "eps"), ("eps", float("nan"), ss.INVALID_ARGUMENT, "eps"),
                 ("eps", float("inf"), ss.INVALID_ARGUMENT, "eps"), ("q_ld", 255, ss.INVALID_ARGUMENT, "q_ld"),
                 ("q_out_ld", 255, ss.INVALID_ARGUMENT, "q_out_ld"), ("k_ld", 127, ss.INVALID_ARGUMENT, "k_ld"),
                 ("v_ld", 127, ss.INVALID_ARGUMENT, "v_ld"), ("q", None, ss.INVALID_ARGUMENT, "required"),
                 ("k", None, ss.INVALID_ARGUMENT, "required"), ("v", None, ss.INVALID_ARGUMENT, "required"),
                 ("q_out", None, ss.INVALID_ARGUMENT, "required"), ("inv_freq", None, ss.INVALID_ARGUMENT, "inv_freq")]


def refused(lib, fn, op, r, c, status, needle):
    assert fn(None, ctypes.byref(op), ctypes.byref(r), ctypes.byref(c), None) == status
    assert needle in lib.ssb_last_error().decode()


@pytest.mark.parametrize("field,value,status,needle", BAD_CACHE)
def test_bad_caches(lib, field, value, status, needle):
    refused(lib, lib.ssb_attend_rows, attend(), rows(), cache(**{field: value}), status, needle)
    refused(lib, lib.ssb_norm_rope_append, norm_rope(), rows(), cache(**{field: value}), status, needle)


@pytest.mark.parametrize("field,value,status,needle", BAD_ROWS)
def test_bad_rows(lib, field, value, status, needle):
    refused(lib, lib.ssb_attend_rows, attend(), rows(**{field: value}), cache(), status, needle)
    refused(lib, lib.ssb_norm_rope_append, norm_rope(), rows(**{field: value}), cache(), status, needle)


@pytest.mark.parametrize("field,value,status,needle", BAD_ATTEND)
def test_bad_attend(lib, field, value, status, needle):
    refused(lib, lib.ssb_attend_rows, attend(**{field: value}), rows(), cache(), status, needle)


@pytest.mark.parametrize("field,value,status,needle", BAD_NORM_ROPE)
def test_bad_norm_rope(lib, field, value, status, needle):
    refused(lib, lib.ssb_norm_rope_append, norm_rope(**{field: value}), rows(), cache(), status, needle)


def test_null_structs_and_context(lib):
    a, n, r, c = attend(), norm_rope(), rows(), cache()
    for fn, op in ((lib.ssb_attend_rows, a), (lib.ssb_norm_rope_append, n)):
        for args in ((None, r, c), (op, None, c), (op, r, None)):
            assert fn(None, *[None if x is None else ctypes.byref(x) for x in args], None) == ss.INVALID_ARGUMENT
            assert "null" in lib.ssb_last_error().decode()
        refused(lib, fn, op, r, c, ss.INVALID_ARGUMENT, "ctx")


def test_the_binding_checks_its_tensors():
    torch = pytest.importorskip("torch")
    k = torch.zeros(3, 16, 2, 64)
    table = torch.zeros(2, 4, dtype=torch.int32)
    c = ss.KvCache(k, k.clone(), table)
    assert (c.struct.pages, c.struct.page_size, c.struct.kv_heads, c.struct.head_dim) == (3, 16, 2, 64)
    assert (c.struct.page_stride, c.struct.position_stride, c.struct.head_stride) == (2048, 128, 64)
    length = torch.zeros(2, dtype=torch.int32)
    c.rows(2, length, None, 1, None)
    for bad in (lambda: ss.KvCache(k, k[:2], table), lambda: ss.KvCache(k, k.transpose(1, 2).contiguous().transpose(1, 2), table),
                lambda: ss.KvCache(k, k.bfloat16(), table), lambda: ss.KvCache(k, k, table.long()), lambda: ss.KvCache(k, k, table[0]),
                lambda: ss.KvCache(k[..., ::2], k[..., ::2], table), lambda: c.rows(2, length.long(), None, 1, None),
                lambda: c.rows(2, length[:1], None, 1, None), lambda: c.rows(2, length, length, 1, None),
                lambda: c.rows(2, length, None, 1, torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ss.KvCache(k.half(), k.half(), table)
    rows = torch.zeros(5, 4, 64)
    assert c.check_heads("q", rows, torch.float32, 4, 5) == 256 and c.check_heads("q", rows[:1], torch.float32, 0, -1) == 256
    assert c.check_heads("q", torch.zeros(5, 300)[:, :256].view(5, 4, 64), torch.float32, 4, 5) == 300
    for bad in (rows[0], rows.bfloat16(), rows[..., :32], rows[:, ::2], rows.transpose(1, 2).contiguous().transpose(1, 2), rows[:4]):
        with pytest.raises(ValueError):
            c.check_heads("q", bad, torch.float32, 4, 5)
    for bad in (torch.zeros(64).double(), torch.zeros(32), torch.zeros(128)[::2]):
        with pytest.raises(ValueError):
            c.check_weight("q_weight", bad)


def test_a_number_too_large_for_its_field():
    torch = pytest.importorskip("torch")
    k = torch.zeros(3, 16, 2, 64)
    c, length, q = ss.KvCache(k, k.clone(), torch.zeros(2, 4, dtype=torch.int32)), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, 64)
    s = ss.Sampler.__new__(ss.Sampler)  # refused before the library is called
    s.ctx = s.lib = None
    for bad in (dict(window=1 << 31), dict(sinks=-(1 << 31) - 1), dict(max_length=1 << 32), dict(max_rows=1 << 31)):
        with pytest.raises(ValueError, match="does not fit"):
            s.attend(q, c, length, **{"scale": 0.125, "max_rows": 1, **bad})
    freq = torch.ones(32, dtype=torch.float64)
    with pytest.raises(ValueError, match="does not fit"):
        s.norm_rope_append(q, q[:, :2], q[:, 2:], c, length, freq, max_rows=1 << 31)
    # a scale beyond 32 bits becomes infinite, as in C, and is refused by the library (test_bad_attend)
    assert ss._PACK_ATTEND.unpack(ss._packed(ss._PACK_ATTEND, *[0] * 4, 1e300, *[0] * 8))[4] == float("inf")


def test_tensors_of_another_device_are_refused():
    """The binding refuses a cache that is not on its engine's device (CPU tensors among them) before the library is called."""
    torch = pytest.importorskip("torch")
    k = torch.zeros(3, 16, 2, 64)
    c, length, q = ss.KvCache(k, k.clone(), torch.zeros(2, 4, dtype=torch.int32)), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, 64)
    freq = torch.ones(32, dtype=torch.float64)
    s = ss.Sampler.__new__(ss.Sampler)
    s.ctx = s.lib = None  # a call would fail on these
    for device in (0, 1):
        s.device = device
        with pytest.raises(ValueError, match=f"cuda:{device}"):
            s.attend(q, c, length, 0.125)
        with pytest.raises(ValueError, match=f"cuda:{device}"):
            s.norm_rope_append(q, q[:, :2], q[:, 2:], c, length, freq)
