"""Row scores and the fitting step without a GPU: refusals of CPU tensors and the C entry points'
checks of their arguments (made on the host before any launch)."""

import ctypes

import pytest
import torch

from kbench_b200 import _lib, fitting, scoring


def _lib_or_skip():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libkb_solver.so not built")
    return _lib.lib()


def test_cpu_tensors_are_refused():
    x = torch.zeros((2, 3))
    for call in (lambda: scoring.score_rows(x), lambda: scoring.score_rows_backward(x, x, x),
                 lambda: fitting.gradient_norm([x]), lambda: fitting.clip_gradients([x], 1.0),
                 lambda: fitting.adam_step([x], [x], [x], [x], 1, lr=0.1)):
        with pytest.raises(RuntimeError):
            call()


def test_score_entry_points_check_their_arguments():
    lib = _lib_or_skip()
    some = ctypes.c_void_p(4096)  # never dereferenced: every call is refused, or has no rows

    def score(stride=8, dtype=0, rows=2, cols=8, given=0, top=0, ptr=some):
        return lib.kb_score_rows(some, stride, dtype, rows, cols, 0, None, given, top, ptr, some, None, None, None, some,
                                 None)

    assert score(rows=0) == _lib.KB_OK
    for bad in ({"rows": -1}, {"cols": -1}, {"stride": -8}, {"dtype": 3}, {"dtype": -1}, {"given": 1}, {"given": 33},
                {"top": 1}, {"top": 33}, {"ptr": None}):
        assert score(**bad) == _lib.KB_ERR_ARG, bad
    assert score(rows=1 << 31) == _lib.KB_ERR_SIZE
    assert score(cols=(1 << 30) + 1) == _lib.KB_ERR_SIZE

    def grad(stride=8, dtype=0, rows=2, cols=8, stats=some, gg=None, out=some, out_stride=8, ge=None, given=0):
        return lib.kb_score_rows_backward(some, stride, dtype, rows, cols, 0, stats, None, None, given, None, gg, ge, out,
                                          out_stride, None)

    assert grad(rows=0) == _lib.KB_OK and grad(cols=0) == _lib.KB_OK
    for bad in ({"rows": -1}, {"stats": None}, {"out": None}, {"out_stride": 7}, {"ge": some}, {"gg": some, "given": 1},
                {"dtype": 7}, {"given": 33}):
        assert grad(**bad) == _lib.KB_ERR_ARG, bad


def test_fit_entry_points_check_their_arguments():
    lib = _lib_or_skip()
    size = ctypes.c_longlong()
    assert lib.kb_fit_workspace(-1, ctypes.byref(size)) == _lib.KB_ERR_ARG
    assert lib.kb_fit_workspace(3, None) == _lib.KB_ERR_ARG
    assert lib.kb_fit_workspace(1, ctypes.byref(size)) == _lib.KB_OK
    small = size.value
    assert lib.kb_fit_workspace(5000, ctypes.byref(size)) == _lib.KB_OK and size.value > small > 0
    some = ctypes.c_void_p(4096)
    one = (ctypes.c_longlong * 1)

    def clip(ptr=4096, count=4, dtype=0, n=1, kind=2, norm=some, max_norm=1.0, ws=some, ws_bytes=small):
        return lib.kb_clip_gradients(one(ptr), one(ptr), one(count), (ctypes.c_int * 1)(dtype), n, kind, max_norm, norm,
                                     ws, ws_bytes, None)

    for bad in ({"ptr": 0}, {"ptr": 4098}, {"count": -1}, {"dtype": 3}, {"n": -1}, {"kind": 1}, {"norm": None},
                {"ws": None}, {"ws_bytes": 8}, {"max_norm": -1.0}, {"max_norm": float("nan")}):
        assert clip(**bad) == _lib.KB_ERR_ARG, bad

    def adam(p=4096, c1=0.1, c2=0.1, kind=-1, max_norm=1.0, norm=some, ws_bytes=small):
        return lib.kb_adam_step(one(p), one(4096), one(4096), one(4096), one(4), (ctypes.c_int * 1)(1), 1, 0.1, 0.9, 0.9,
                                1e-8, 0.0, c1, c2, kind, max_norm, norm, some, ws_bytes, None)

    for bad in ({"p": 0}, {"p": 4098}, {"c1": 0.0}, {"c2": -1.0}, {"kind": 1}, {"kind": 2, "max_norm": -2.0},
                {"kind": 2, "norm": None}, {"ws_bytes": 0}):
        assert adam(**bad) == _lib.KB_ERR_ARG, bad


def _host_or_skip():
    try:
        return _lib.host()
    except RuntimeError:
        pytest.skip("_kb_host.so not built")


def test_overlap_finds_shared_memory():
    """Random placements in one buffer, in random order, against comparing every pair."""
    host = _host_or_skip()
    g = torch.Generator().manual_seed(0)
    flat = torch.zeros(4000)
    for trial in range(300):
        n_w, n_r = (int(torch.randint(0, 7, (1,), generator=g)) for _ in range(2))
        spans = [(int(torch.randint(0, 3900, (1,), generator=g)), int(torch.randint(0, 90, (1,), generator=g)))
                 for _ in range(n_w + n_r)]
        if trial % 3 == 0:
            spans[n_w:] = [spans[i] if i < n_w else s for i, s in enumerate(spans[n_w:])]
        ts = [flat[a:a + m] for a, m in spans]
        w, r = ts[:n_w], ts[n_w:]

        def meet(x, y):
            return x[1] > 0 and y[1] > 0 and x[0] < y[0] + y[1] and y[0] < x[0] + x[1]

        sw, sr = spans[:n_w], spans[n_w:]
        for in_place in (False, True):
            want = any(meet(sw[i], sw[j]) for i in range(n_w) for j in range(i)) or any(
                meet(x, y) and not (in_place and i == j and x == y) for i, x in enumerate(sw) for j, y in enumerate(sr))
            assert host.overlap(w, r, in_place) == want, (sw, sr, in_place)


def test_lists_are_described():
    host = _host_or_skip()
    ts = [torch.zeros(3, 4), torch.zeros(0), torch.zeros(5).bfloat16()]
    for other, want in (([t.clone() for t in ts], True), (ts[:2], False), ([torch.zeros(4, 3), ts[1], ts[2]], False)):
        described, flags, same, _ = host.gather((ts, other), 0, 0, False)
        assert same == want and len(described) == 3 and len(flags) == 2
    addresses, dtypes = described[0]
    assert len(addresses) == 24 and len(dtypes) == 12 and len(described[2]) == 24 and flags[0] & 1  # not on a GPU
    for bad in ((ts, (1, 2)), ([torch.zeros(2), None],), ("ab",)):
        with pytest.raises(TypeError):
            host.gather(bad, 0, 0, False)
    with pytest.raises(TypeError):
        host.gather(ts, 0, 0, False)


def test_written_tensors_get_a_new_version():
    host = _host_or_skip()
    a, b = torch.zeros(3), torch.zeros(4)
    with torch.inference_mode():
        c = torch.zeros(2)
    host.written([a, c, b[1:]])  # a view's version is its base's; inference tensors have none
    assert a._version == 1 and b._version == 1
    with pytest.raises(TypeError):
        host.written([a, None])


def test_a_new_version_is_looked_at_again():
    from types import SimpleNamespace

    from kbench_b200 import glue
    host = _host_or_skip()
    static, w = SimpleNamespace(), torch.zeros(5)
    assert glue.col_weights_uniform_for(static, w)
    ctypes.c_float.from_address(w.data_ptr()).value = 1.0
    host.written([w])
    assert not glue.col_weights_uniform_for(static, w)


def test_rows_past_the_longest_are_refused():
    """Before a 32-bit argument can drop the upper bits of a row's length."""
    from types import SimpleNamespace
    for S in ((1 << 30) + 1, 1 << 32, (1 << 32) + 5):
        rows = SimpleNamespace(device=SimpleNamespace(type="cuda"), dtype=torch.bfloat16, ndim=2, shape=(1, S),
                               stride=lambda d: 1)
        with pytest.raises(ValueError):
            scoring._check_rows("score_rows", rows)
    text = _lib.HEADER.read_text()
    assert f"#define KB_MAX_SCORE_COLS {scoring.MAX_COLS}\n" in text


def test_shared_memory_is_seen_through_other_storages():
    flat = torch.zeros(100)
    rows = flat[:60].view(6, 10)
    same = torch.from_dlpack(flat[30:90]).view(6, 10)
    assert same.untyped_storage().data_ptr() != rows.untyped_storage().data_ptr()
    assert scoring._overlap(same, rows) and not scoring._overlap(torch.from_dlpack(flat[60:]).view(4, 10), rows)


def test_addresses_off_their_types_boundary_are_refused():
    """Such an access would fault on the device."""
    lib = _lib_or_skip()
    p = {"rows": 4096, "given": 4096, "mass": 4096, "entropy": 4096, "glp": 4096, "tlp": 4096, "tcol": 4096, "stats": 4096}
    for dtype, off in ((0, {"rows": 4098}), (1, {"rows": 4097}), (2, {"rows": 4099}), (0, {"given": 4100}),
                       (0, {"mass": 4098}), (0, {"entropy": 4097}), (0, {"glp": 4098}), (0, {"tlp": 4098}),
                       (0, {"tcol": 4100}), (0, {"stats": 4098})):
        a = dict(p, **off)
        assert lib.kb_score_rows(a["rows"], 8, dtype, 2, 8, 0, a["given"], 1, 1, a["mass"], a["entropy"], a["glp"],
                                 a["tlp"], a["tcol"], a["stats"], None) == _lib.KB_ERR_ARG, off
    p = {"rows": 4096, "stats": 4096, "entropy": 4096, "given": 4096, "gm": 4096, "gg": 4096, "ge": 4096, "out": 8192}
    for dtype, off in ((0, {"rows": 4098}), (1, {"rows": 4097}), (1, {"out": 8193}), (0, {"out": 8194}), (0, {"given": 4100}),
                       (0, {"stats": 4098}), (0, {"entropy": 4098}), (0, {"gm": 4098}), (0, {"gg": 4098}), (0, {"ge": 4098})):
        a = dict(p, **off)
        assert lib.kb_score_rows_backward(a["rows"], 8, dtype, 2, 8, 0, a["stats"], a["entropy"], a["given"], 1, a["gm"],
                                          a["gg"], a["ge"], a["out"], 8, None) == _lib.KB_ERR_ARG, off
    size = ctypes.c_longlong()
    lib.kb_fit_workspace(1, ctypes.byref(size))
    one, dtypes = (ctypes.c_longlong * 1), (ctypes.c_int * 1)(0)
    for ws, norm in ((4104, 4096), (4096, 4098)):
        assert lib.kb_clip_gradients(one(4096), one(4096), one(4), dtypes, 1, 2, 1.0, norm, ws, size.value,
                                     None) == _lib.KB_ERR_ARG
        assert lib.kb_adam_step(one(4096), one(4096), one(4096), one(4096), one(4), dtypes, 1, 0.1, 0.9, 0.9, 1e-8, 0.0, 0.1,
                                0.1, 2, 1.0, norm, ws, size.value, None) == _lib.KB_ERR_ARG


def test_strides_of_dimensions_of_one_do_not_matter():
    a = torch.zeros(5 * 3).as_strided((3, 1, 5), (1, 99, 3))
    b = torch.zeros(5 * 3).as_strided((3, 1, 5), (1, 15, 3))
    assert fitting._dense(a) and fitting._same_layout(a, b) and not fitting._same_layout(a, torch.zeros(3, 1, 5))
