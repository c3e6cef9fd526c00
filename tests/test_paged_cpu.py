"""Refusals of the operators over a caller's paged K/V cache: arguments are checked before the handle, so no GPU is needed."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def api(built_lib):
    from mini_llm_cuda_b200 import api as _api
    return _api


def cache(api, **kw):
    d = dict(kpool=4096, vpool=8192, kscale=None, vscale=None, page_table=64, pt_stride=4, num_pages=9, kv_heads=2, head_dim=64,
             dtype=api.DT_BF16, k_scale=1.0, v_scale=1.0)
    d.update(kw)
    return api.PagedKvStruct(**d)


def new_rows(api, **kw):
    d = dict(row_start=None, kv_lens=128, batch=3, rows=3, max_rows=0)
    d.update(kw)
    return api.NewRowsStruct(**d)


def calls(api, kv, rows, dt=None, ptr=1 << 20, stride=1 << 10):
    """Status of each operator with these descriptions and no handle."""
    L, dt = api.lib(), api.DT_BF16 if dt is None else dt
    kvp, rp = C.byref(kv) if kv is not None else None, C.byref(rows) if rows is not None else None
    return [L.mlb_op_kv_append(None, kvp, rp, dt, ptr, stride, ptr, stride, None, 0, None, 0, None, 0, 0, None),
            L.mlb_op_kv_read(None, kvp, rp, dt, ptr, stride, ptr, stride, None),
            L.mlb_op_attn_paged(None, kvp, rp, dt, ptr, stride, None, ptr, stride, 4, 0.0, 0, 0, None)]


def test_without_a_handle(api):
    assert calls(api, cache(api), new_rows(api)) == [api.MLB_E_INVALID] * 3
    assert b"null handle" in api.lib().mlb_last_error()
    assert calls(api, None, new_rows(api)) == [api.MLB_E_INVALID] * 3
    assert calls(api, cache(api), None) == [api.MLB_E_INVALID] * 3
    assert api.lib().mlb_ops_status(None, None) == api.MLB_E_INVALID
    assert api.lib().mlb_ops_new(0, None) == api.MLB_E_INVALID
    api.lib().mlb_ops_free(None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(kpool=None), "INVALID", b"null pointer"),
    (dict(page_table=None), "INVALID", b"null pointer"),
    (dict(dtype=3), "INVALID", b"float32, bfloat16 or fp4"),
    (dict(dtype=0), "INVALID", b"float32, bfloat16 or fp4"),
    (dict(dtype=4), "INVALID", b"has scales"),
    (dict(dtype=4, kscale=256, vscale=512, k_scale=0.0), "INVALID", b"positive"),
    (dict(dtype=4, kscale=256, vscale=512, v_scale=float("nan")), "INVALID", b"positive"),
    (dict(dtype=4, kscale=256, vscale=512, v_scale=float("inf")), "INVALID", b"positive"),
    (dict(dtype=4, kscale=257, vscale=512), "INVALID", b"16 bytes"),
    (dict(kpool=4104), "INVALID", b"16 bytes"),
    (dict(pt_stride=0), "INVALID", b">= 1"),
    (dict(pt_stride=1 << 27), "UNSUPPORTED", b"pt_stride"),
    (dict(num_pages=0), "INVALID", b">= 1"),
    (dict(kv_heads=0), "INVALID", b">= 1"),
    (dict(head_dim=96), "UNSUPPORTED", b"64 or 128"),
])
def test_refused_caches(api, kw, status, text):
    want = getattr(api, "MLB_E_" + status)
    assert calls(api, cache(api, **kw), new_rows(api)) == [want] * 3
    assert text in api.lib().mlb_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(kv_lens=None), "INVALID"), (dict(batch=0), "INVALID"), (dict(batch=4097), "INVALID"), (dict(rows=-1), "INVALID"),
    (dict(max_rows=-1), "INVALID"), (dict(rows=1 << 30), "UNSUPPORTED"),
])
def test_refused_rows(api, kw, status):
    assert calls(api, cache(api), new_rows(api, **kw)) == [getattr(api, "MLB_E_" + status)] * 3


def test_refused_row_tensors(api):
    kv, rows = cache(api), new_rows(api)
    assert calls(api, kv, rows, dt=api.DT_FP8) == [api.MLB_E_INVALID] * 3
    assert calls(api, kv, rows, ptr=None) == [api.MLB_E_INVALID] * 3
    assert calls(api, kv, rows, ptr=(1 << 20) + 1) == [api.MLB_E_INVALID] * 3
    assert calls(api, kv, rows, stride=127) == [api.MLB_E_INVALID] * 3
    assert b"stride" in api.lib().mlb_last_error()
    # no rows: nothing is looked at but the handle
    assert calls(api, kv, new_rows(api, rows=0), ptr=None) == [api.MLB_E_INVALID] * 3
    assert b"null handle" in api.lib().mlb_last_error()


def test_refused_attention(api):
    L, kv, rows, p = api.lib(), cache(api), new_rows(api), 1 << 20

    def status(heads=4, scale=0.0, window=0, sinks=0, gate=None):
        return L.mlb_op_attn_paged(None, C.byref(kv), C.byref(rows), api.DT_BF16, p, 4096, gate, p, 4096, heads, scale, window, sinks, None)

    assert status(heads=3) == api.MLB_E_INVALID
    assert status(heads=0) == api.MLB_E_INVALID
    assert status(heads=18) == api.MLB_E_UNSUPPORTED
    for kw in (dict(window=-1), dict(sinks=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(gate=2)):
        assert status(**kw) == api.MLB_E_INVALID
        assert b"null handle" not in L.mlb_last_error()


def test_refused_append(api):
    L, kv, rows, p = api.lib(), cache(api), new_rows(api), 1 << 20

    def status(rope=None, rope_len=0, q=None, q_out=None, heads=0):
        return L.mlb_op_kv_append(None, C.byref(kv), C.byref(rows), api.DT_BF16, p, 4096, p, 4096, rope, rope_len, q, 4096, q_out, 4096, heads, None)

    for kw in (dict(rope=4096, rope_len=0), dict(rope=4097, rope_len=5), dict(q=p, q_out=None, heads=4), dict(q=p, q_out=p, heads=0),
               dict(q=p, q_out=p + 1, heads=4)):
        assert status(**kw) == api.MLB_E_INVALID
        assert b"null handle" not in L.mlb_last_error()


def test_no_device(api):
    import torch
    if torch.cuda.is_available():
        pytest.skip("this machine has a GPU")
    h = C.c_void_p()
    assert api.lib().mlb_ops_new(0, C.byref(h)) == api.MLB_E_CUDA
    assert not h.value


def test_refused_head_counts(api):
    assert calls(api, cache(api, kv_heads=65536), new_rows(api), stride=1 << 24) == [api.MLB_E_UNSUPPORTED] * 3
    L, kv, rows, p = api.lib(), cache(api), new_rows(api), 1 << 20
    assert L.mlb_op_kv_append(None, C.byref(kv), C.byref(rows), api.DT_BF16, p, 4096, p, 4096, None, 0, p, 1 << 30, p, 1 << 30, 8 * 65535 + 1, None) \
        == api.MLB_E_UNSUPPORTED


def test_refused_pools_of_too_many_rows(api):
    """A row of a bf16 pool is a coordinate of a tensor map where prompts may come; pools of 4 bits and steps have no such limit."""
    L, p = api.lib(), 1 << 20

    def status(dtype=api.DT_BF16, row_start=64, max_rows=0, pages=(1 << 26) + 1, rows=200):
        kv = cache(api, dtype=dtype, num_pages=pages, kscale=256, vscale=512)
        nr = new_rows(api, row_start=row_start, rows=rows, max_rows=max_rows)
        rc = L.mlb_op_attn_paged(None, C.byref(kv), C.byref(nr), api.DT_BF16, p, 4096, None, p, 4096, 4, 0.0, 0, 0, None)
        return rc, b"2^31" in L.mlb_last_error()

    assert status() == (api.MLB_E_UNSUPPORTED, True)
    for kw in (dict(dtype=api.DT_FP4), dict(row_start=None), dict(max_rows=16), dict(rows=16), dict(pages=(1 << 26) - 1)):
        assert status(**kw) == (api.MLB_E_INVALID, False)    # (no handle)


class FakeTensor:
    """As much of a CUDA tensor as the calls look at."""

    def __init__(self, dtype, rows, width):
        import torch
        self.dtype, self.shape, self._stride = dtype, torch.Size((rows, width)), (width, 1)

    def get_device(self):
        return 0

    def stride(self, i=None):
        return self._stride if i is None else self._stride[i]

    def data_ptr(self):
        return 1 << 20


@pytest.fixture
def fake_ops(api, monkeypatch):
    """api.Ops whose calls end in a list instead of the library, on a device whose current torch stream is 4711."""
    import types
    import torch
    ops, calls = api.Ops.__new__(api.Ops), []
    ops._h, ops.device = C.c_void_p(), 0
    ops._append = ops._read = ops._attn = lambda *a: calls.append(a) or 0
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=4711) if device == 0 else None)
    cache = types.SimpleNamespace(batch=3, device=0, width=128, head_dim=64, ref=None)
    rows = types.SimpleNamespace(batch=3, device=0, rows=5, ref=None)
    return ops, calls, cache, rows


def test_torch_current_stream_unless_told(api, fake_ops, monkeypatch):
    """A call without a stream runs behind what torch has on its current one."""
    import types
    import torch
    ops, calls, cache, rows = fake_ops
    x, y = FakeTensor(torch.bfloat16, 5, 128), FakeTensor(torch.bfloat16, 5, 256)
    fake = types.SimpleNamespace(mlb_ops_status=lambda h, stream: calls.append((stream,)) or 0)
    monkeypatch.setattr(api, "lib", lambda: fake)
    for kw, want in ((dict(), 4711), (dict(stream=0), 0), (dict(stream=5), 5)):
        ops.kv_append(cache, rows, x, x, **kw)
        ops.kv_read(cache, rows, x, x, **kw)
        ops.attn_paged(cache, rows, y, y, heads=4, **kw)
        ops.status(*kw.values())
        assert [c[-1] for c in calls] == [want] * 4
        calls.clear()


def test_refused_rotation_in_place_with_another_stride(api):
    """Row i of q_out over row j of q: rotated and not rotated rows in each other's place."""
    L, kv, rows, p = api.lib(), cache(api), new_rows(api), 1 << 20

    def status(q_stride, out_stride, rows=rows):
        rc = L.mlb_op_kv_append(None, C.byref(kv), C.byref(rows), api.DT_BF16, p, 4096, p, 4096, None, 0, p, q_stride, p, out_stride, 4, None)
        return rc, b"same stride" in L.mlb_last_error()

    assert status(4096, 512) == (api.MLB_E_INVALID, True)
    assert status(4096, 4096) == (api.MLB_E_INVALID, False)              # (no handle)
    assert status(4096, 512, new_rows(api, batch=1, rows=1)) == (api.MLB_E_INVALID, False)


def test_numbers_beyond_32_bits(api, fake_ops):
    """A window, a count of first positions or a most of rows above 2^31 is one that nothing reaches, and not its low 32 bits."""
    import torch
    ops, calls, cache, rows = fake_ops
    y = FakeTensor(torch.bfloat16, 5, 256)
    top = (1 << 31) - 1
    for window, sinks, want in ((5, 3, (5, 3)), ((1 << 32) + 5, 1 << 32, (top, top)), (top + 1, 0, (top, 0)), (-(1 << 32), 4, (-1, 4)), (0, -(1 << 33) - 7, (0, -1))):
        ops.attn_paged(cache, rows, y, y, heads=4, window=window, sinks=sinks)
        assert calls.pop()[-3:-1] == want
    lens = FakeTensor(torch.int32, 1, 3)
    lens.is_cuda, lens.is_contiguous, lens.numel = True, lambda: True, lambda: 3
    assert api.NewRows(lens, 3, max_rows=(1 << 32) + 1).struct.max_rows == top
    assert api.NewRows(lens, 3, max_rows=7).struct.max_rows == 7


def test_rows_of_one_head(api, fake_ops):
    """[rows][1][head_dim] has no second head, so the stride to it says nothing; of more heads it has to be dense."""
    import torch
    ops, calls, cache, rows = fake_ops

    def rows_of(shape, strides):
        x = FakeTensor(torch.float32, 5, 128)
        x.shape, x._stride = torch.Size(shape), strides
        return ops._rows(x, "k", (5, 128), torch.float32)

    assert rows_of((5, 1, 128), (128, 640, 1)) == (1 << 20, 128)
    assert rows_of((5, 2, 64), (200, 64, 1)) == (1 << 20, 200)
    for shape, strides in (((5, 2, 64), (64, 320, 1)), ((5, 1, 128), (128, 640, 2)), ((5, 1, 64), (64, 320, 1)), ((4, 1, 128), (128, 640, 1))):
        with pytest.raises(ValueError):
            rows_of(shape, strides)
