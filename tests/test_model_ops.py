"""Host-side checks of the operators of language models: sizes, layouts and refusals that are
decided before any device work."""
import ctypes

import pytest
import torch


def _mat(dcopy, data=0x10000, rows=4, cols=8, pitch=8, code=0):
    return ctypes.byref(dcopy.DcopyMatrix(data, rows, cols, pitch, code, 0))


def test_expert_rows(dcopy):
    assert dcopy.expert_rows(100, 8, 1) == 100
    assert dcopy.expert_rows(100, 8, 16) == 220
    assert dcopy.expert_rows(3, 8, 16) == 48  # at most 3 experts hold anything
    assert dcopy.expert_rows(0, 8, 16) == 0
    for args, code in (((-1, 8, 1), dcopy.ERR_PARAM_INVALID), ((1, 0, 1), dcopy.ERR_PARAM_INVALID),
                       ((1, 8, 0), dcopy.ERR_PARAM_INVALID),
                       ((1 << 31, 8, 1), dcopy.ERR_SHAPE_INVALID),
                       (((1 << 31) - 1, 8, 2), dcopy.ERR_SHAPE_INVALID)):
        with pytest.raises(dcopy.DcopyError) as e:
            dcopy.expert_rows(*args)
        assert e.value.code == code


def test_workspaces_grow_with_their_arguments(dcopy):
    a, b = dcopy.embedding_grad_workspace(1000, 50, 64), dcopy.embedding_grad_workspace(2000, 50, 64)
    assert 0 < a < b
    assert dcopy.expert_sort_workspace(1 << 20, 64) > dcopy.expert_sort_workspace(1 << 10, 64) > 0
    for f, args in ((dcopy.embedding_grad_workspace, (-1, 5, 5)),
                    (dcopy.embedding_grad_workspace, (1, 1 << 31, 5)),
                    (dcopy.expert_sort_workspace, (5, 0))):
        with pytest.raises(dcopy.DcopyError) as e:
            f(*args)
        assert e.value.code == dcopy.ERR_PARAM_INVALID
    with pytest.raises(dcopy.DcopyError) as e:
        dcopy.expert_sort_workspace(5, 1024)
    assert e.value.code == dcopy.ERR_UNSUPPORTED


@pytest.mark.parametrize("change,code", [
    (dict(code=11), "ERR_DATATYPE_INVALID"), (dict(rows=-1), "ERR_SHAPE_INVALID"),
    (dict(cols=1 << 31), "ERR_SHAPE_INVALID"), (dict(pitch=7), "ERR_PARAM_INVALID"),
    (dict(data=0x10002), "ERR_PARAM_INVALID"), (dict(data=None), "ERR_PARAM_INVALID"),
    (dict(pitch=1 << 62), "ERR_PARAM_INVALID"),
])
def test_matrix_checks(dcopy, change, code):
    """Each bad field of a matrix is refused with its status."""
    lib = dcopy.lib()
    ids = _mat(dcopy, 0x40000, 4, 1, 1, 9)
    rc = lib.dcopy_embedding_lookup(_mat(dcopy, **change), _mat(dcopy), ids, 0, 1.0, None)
    assert rc == getattr(dcopy, code), lib.dcopy_last_error_message()


def test_null_arguments(dcopy):
    lib, m = dcopy.lib(), _mat(dcopy)
    assert lib.dcopy_embedding_lookup(None, m, m, 0, 1.0, None) == dcopy.ERR_PARAM_INVALID
    assert lib.dcopy_embedding_grad(m, None, m, 0, 1.0, 0, None, 0, None) == dcopy.ERR_PARAM_INVALID
    assert lib.dcopy_expert_sort(None, None, 0, None, None, 4, 1, None, 0, None) == dcopy.ERR_PARAM_INVALID
    assert lib.dcopy_expert_dispatch(m, None, None, 1, None, None, None) == dcopy.ERR_PARAM_INVALID
    assert lib.dcopy_expert_combine(None, m, None, 1, None, None) == dcopy.ERR_PARAM_INVALID
    assert lib.dcopy_expert_combine_grad(m, m, m, m, None, 1, None, None, None) == dcopy.ERR_PARAM_INVALID
    assert lib.dcopy_grad_list_build(None, None, 0, None, 0, None) == dcopy.ERR_PARAM_INVALID
    assert lib.dcopy_clip_grad_norm(None, 1.0, 1e-6, None, None) == dcopy.ERR_PARAM_INVALID
    empty = dcopy.DcopyGradList()
    assert lib.dcopy_grad_sum_squares(ctypes.byref(empty), None, None) == dcopy.ERR_PARAM_INVALID
    for bound in (float("nan"), -1.0):
        assert lib.dcopy_clip_grad_norm(ctypes.byref(empty), bound, 0.0, None, None) == \
            dcopy.ERR_PARAM_INVALID


def test_python_refuses_host_tensors(dcopy):
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError):
        dcopy.embedding_lookup(x, x, ids)
    with pytest.raises(ValueError):
        dcopy.expert_dispatch(x, x, ids)
    with pytest.raises(ValueError):
        dcopy.GradList([x])
    with pytest.raises(ValueError):
        dcopy.GradList([])


def test_layout_of_a_tensor(dcopy):
    """Rows, columns, pitch and type that a call reads from a tensor's shape and strides."""
    from dcopy import model_ops

    def read(t):
        return model_ops._calls.layout(t)

    x = torch.zeros(6, 10, 16)
    assert read(x) == (60, 16, 16, 0)
    assert read(x[:, :, :8]) == (60, 8, 16, 0)
    assert read(x[:, 3]) == (6, 16, 160, 0)
    assert read(x[0]) == (10, 16, 16, 0)
    assert read(x[2:3, 4:5]) == (1, 16, 16, 0)
    assert read(torch.zeros(1, 5, 1, 7, dtype=torch.bfloat16)) == (5, 7, 7, 27)
    assert read(torch.zeros(12, dtype=torch.int64)) == (1, 12, 0, 9)
    assert read(torch.zeros(12, dtype=torch.int32)[::3]) == (4, 1, 3, 3)
    assert read(torch.zeros(9, 1)) == (9, 1, 1, 0)
    assert read(torch.zeros(3, 4, dtype=torch.float64)) == (3, 4, 4, -1)
    for bad in (x[:, :5],                       # two row pitches
                torch.zeros(4, 6).t(),          # columns that are not dense
                torch.zeros(1).expand(5)):      # one element for all
        with pytest.raises(ValueError):
            read(bad)
    with pytest.raises(ValueError):
        read([1, 2])


def test_records_match_the_c_abi(dcopy, tmp_path, monkeypatch):
    import test_abi_layout as layout
    monkeypatch.setattr(layout, "STRUCTS", {
        "DcopyMatrix": ["data", "rows", "cols", "pitch", "type", "reserved"],
        "DcopyGrad": ["src", "dst", "count", "src_type", "dst_type"],
        "DcopyGradList": ["workspace", "first"],
    })
    layout.test_ctypes_records_match_the_c_abi(dcopy, tmp_path)


@pytest.mark.parametrize("spans,fine", [
    ([(0, 0), (400, 400)], True), ([(0, 1000), (400, 1400)], True),
    ([(0, 1000), (0, 2000)], True),           # one gradient, clipped into two places
    ([(0, 0), (0, 0)], False),                # one gradient twice in place
    ([(0, 0), (396, 396)], False), ([(396, 396), (0, 0)], False),
    ([(0, 1000), (1000, 2000)], False),       # an output is the next gradient
    ([(0, 1000), (400, 1004)], False),        # two outputs meet
    ([(0, 1000), (400, 2000), (2396, 3000)], False),
    ([(0, 4)], False),                        # neither in place nor apart
    ([(0, 20000)], False),                    # the output is the workspace
    ([(100000 - 400, 0)], True), ([(0, 4000), (4, 8000), (8, 12000)], True),
])
def test_gradients_of_a_list_lie_apart(dcopy, spans, fine):
    """Outputs overlap no gradient, no other output and not the workspace.  (Addresses only:
    refused before anything is copied; what passes fails here for want of a GPU, if at all.)"""
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    base, size = 0x10000000, 100000
    arr = (dcopy.DcopyGrad * len(spans))(*[(base + s, base + d, 100, 0, 0) for s, d in spans])
    at = 20000 if (0, 20000) in spans else 200000
    rc = dcopy.lib().dcopy_grad_list_build(ctypes.byref(dcopy.DcopyGradList()), arr, len(arr),
                                           base + at, size, None)
    message = dcopy.lib().dcopy_last_error_message()
    assert (rc == dcopy.ERR_PARAM_INVALID and b"overlaps" in message) == (not fine), message


BASE = 0x20000000
PLACES = {  # argument -> (offset, rows, cols, pitch, type code); 64 tokens x 4 slots, 256 rows, 8 experts
    "lookup": dict(out=(0, 64, 32, 32, 0), table=(1 << 20, 100, 32, 32, 0), ids=(2 << 20, 64, 1, 1, 9)),
    "grad": dict(grad=(0, 100, 32, 32, 0), dout=(1 << 20, 64, 32, 32, 0), ids=(2 << 20, 64, 1, 1, 9),
                 workspace=(3 << 20, 1, 0, 0, 4)),  # as many bytes as are needed, here and below
    "sort": dict(dest=(0, 1, 6400, 0, 3), source=(1 << 20, 1, 6400, 0, 3), offsets=(2 << 20, 1, 9, 0, 3),
                 expert_ids=(3 << 20, 1600, 4, 4, 3), workspace=(4 << 20, 1, 0, 0, 4)),
    "dispatch": dict(out=(0, 256, 32, 32, 0), x=(1 << 20, 64, 32, 32, 0), dest=(2 << 20, 1, 256, 0, 3),
                     source=(3 << 20, 1, 256, 0, 3), weights=(4 << 20, 64, 4, 4, 0)),
    "combine": dict(out=(0, 64, 32, 32, 0), y=(1 << 20, 256, 32, 32, 0), dest=(2 << 20, 1, 256, 0, 3),
                    weights=(4 << 20, 64, 4, 4, 0)),
    "combine_grad": dict(dy=(0, 256, 32, 32, 0), dweights=(1 << 20, 64, 4, 4, 0),
                         dout=(2 << 20, 64, 32, 32, 0), y=(3 << 20, 256, 32, 32, 0),
                         dest=(4 << 20, 1, 256, 0, 3), source=(5 << 20, 1, 256, 0, 3),
                         weights=(6 << 20, 64, 4, 4, 0)),
}
WRITTEN = {"lookup": ["out"], "grad": ["grad", "workspace"], "sort": ["dest", "source", "offsets", "workspace"],
           "dispatch": ["out"], "combine": ["out"], "combine_grad": ["dy", "dweights"]}


def places_of(dcopy, op):
    need = {"grad": lambda: dcopy.embedding_grad_workspace(64, 100, 32),
            "sort": lambda: dcopy.expert_sort_workspace(6400, 8)}
    return {k: (at, r, need[op]() if k == "workspace" else c, p, t)
            for k, (at, r, c, p, t) in PLACES[op].items()}


def call_at(dcopy, op, places):
    """Status and message of a call on made-up addresses."""
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    m = {k: dcopy.DcopyMatrix(BASE + at, r, c, p, t, 0) for k, (at, r, c, p, t) in places.items()}
    ref = {k: ctypes.byref(v) for k, v in m.items()}
    raw = {k: v.data for k, v in m.items()}
    lib = dcopy.lib()
    rc = {
        "lookup": lambda: lib.dcopy_embedding_lookup(ref["out"], ref["table"], ref["ids"], 0, 1.0, None),
        "grad": lambda: lib.dcopy_embedding_grad(ref["grad"], ref["dout"], ref["ids"], 0, 1.0, 0,
                                                 raw["workspace"], m["workspace"].cols, None),
        "sort": lambda: lib.dcopy_expert_sort(raw["dest"], raw["source"], m["source"].cols, raw["offsets"],
                                              ref["expert_ids"], 8, 1, raw["workspace"],
                                              m["workspace"].cols, None),
        "dispatch": lambda: lib.dcopy_expert_dispatch(ref["out"], ref["x"], raw["dest"], 4, raw["source"],
                                                      ref["weights"], None),
        "combine": lambda: lib.dcopy_expert_combine(ref["out"], ref["y"], raw["dest"], 4, ref["weights"], None),
        "combine_grad": lambda: lib.dcopy_expert_combine_grad(
            ref["dy"], ref["dweights"], ref["dout"], ref["y"], raw["dest"], 4, raw["source"],
            ref["weights"], None),
    }[op]()
    return rc, lib.dcopy_last_error_message()


def overlaps(dcopy, op, places):
    rc, message = call_at(dcopy, op, places)
    assert rc != dcopy.OK  # no GPU
    return rc == dcopy.ERR_PARAM_INVALID and b"overlap" in message


@pytest.mark.parametrize("op,written,other", [(op, w, o) for op in PLACES for w in WRITTEN[op]
                                              for o in PLACES[op] if o != w])
def test_what_is_written_lies_apart(dcopy, op, written, other):
    """Whatever a call writes overlaps no other argument, at its first byte or its last."""
    places = places_of(dcopy, op)
    assert not overlaps(dcopy, op, places)
    start, rows, cols, pitch, code = places[other]
    wide = {0: 4, 3: 4, 4: 1, 9: 8}
    first, w_rows, w_cols, w_pitch, w_code = places[written]
    last = first + ((w_rows - 1) * w_pitch + w_cols - 1) * wide[w_code]
    for at in (first + 8, last // 8 * 8):
        assert overlaps(dcopy, op, {**places, other: (at, rows, cols, pitch, code)}), at
    end = (last + wide[w_code] + 15) // 16 * 16
    # Behind its last byte, well before the next argument.
    assert not overlaps(dcopy, op, {**places, other: (end, rows, cols, pitch, code)})


def test_what_may_be_in_place(dcopy):
    """The routing written over the choices it is made of, and weights' gradients over the
    weights; neither at another place of the same memory nor in another type."""
    sort, back = places_of(dcopy, "sort"), places_of(dcopy, "combine_grad")
    at = sort["dest"][0]
    assert not overlaps(dcopy, "sort", {**sort, "expert_ids": (at, 1600, 4, 4, 3)})
    assert overlaps(dcopy, "sort", {**sort, "expert_ids": (at, 1600, 4, 5, 3)})
    assert overlaps(dcopy, "sort", {**sort, "expert_ids": (at, 1600, 4, 4, 9)})
    assert overlaps(dcopy, "sort", {**sort, "expert_ids": (at + 4, 1600, 4, 4, 3)})
    at = back["dweights"][0]
    assert not overlaps(dcopy, "combine_grad", {**back, "weights": (at, 64, 4, 4, 0)})
    assert overlaps(dcopy, "combine_grad", {**back, "weights": (at, 64, 4, 5, 0)})
    assert overlaps(dcopy, "combine_grad", {**back, "weights": (at + 4, 64, 4, 4, 0)})


def test_columns_of_one_buffer_lie_apart(dcopy):
    """Rows of one pitch that interleave share no byte."""
    back = places_of(dcopy, "combine_grad")
    dw, w = (1 << 20, 64, 4, 8, 0), ((1 << 20) + 16, 64, 4, 8, 0)
    assert not overlaps(dcopy, "combine_grad", {**back, "dweights": dw, "weights": w})
    assert not overlaps(dcopy, "combine_grad", {**back, "dweights": w, "weights": dw})
    for at in (12, 20, 32 + 12):  # a column shared, behind a slice or before the next row's
        moved = ((1 << 20) + at, 64, 4, 8, 0)
        assert overlaps(dcopy, "combine_grad", {**back, "dweights": dw, "weights": moved})
        assert overlaps(dcopy, "combine_grad", {**back, "dweights": moved, "weights": dw})
    assert overlaps(dcopy, "combine_grad", {**back, "dweights": dw, "weights": (*w[:3], 12, 0)})
    look = places_of(dcopy, "lookup")
    assert not overlaps(dcopy, "lookup", {**look, "out": (0, 64, 32, 64, 0), "table": (128, 100, 32, 64, 0)})
    assert overlaps(dcopy, "lookup", {**look, "out": (0, 64, 32, 64, 0), "table": (124, 100, 32, 64, 0)})


def test_numbers_of_a_clipping_call_lie_apart(dcopy):
    """The sum and the norm lie outside the list's workspace, and the norm outside the sum."""
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    lib, built = dcopy.lib(), dcopy.DcopyGradList()
    built.workspace = BASE

    def refused(rc):
        return rc == dcopy.ERR_PARAM_INVALID and b"overlap" in lib.dcopy_last_error_message()

    ref, far = ctypes.byref(built), BASE + (1 << 20)
    assert refused(lib.dcopy_grad_sum_squares(ref, BASE + 64, None))
    assert refused(lib.dcopy_grad_clip(ref, BASE + 64, 1.0, 0.0, None, None))
    assert refused(lib.dcopy_grad_clip(ref, far, 1.0, 0.0, BASE + 64, None))
    assert refused(lib.dcopy_grad_clip(ref, far, 1.0, 0.0, far + 4, None))
    assert refused(lib.dcopy_clip_grad_norm(ref, 1.0, 0.0, BASE, None))
    assert not refused(lib.dcopy_grad_clip(ref, far, 1.0, 0.0, far + 8, None))


def test_layout_of_an_empty_tensor(dcopy):
    """An empty batch has rows, columns and no pitch to disagree about, wherever its zero is."""
    from dcopy import model_ops

    def read(*shape):
        rows, cols, _, code = model_ops._calls.layout(torch.zeros(*shape))
        assert code == 0
        return rows, cols

    assert read(4, 0, 8) == (0, 8) and read(0, 4, 8) == (0, 8) and read(3, 4, 0, 8) == (0, 8)
    assert read(2, 0, 5, 8) == (0, 8) and read(4, 5, 0) == (20, 0) and read(0) == (1, 0)
    rows, cols, _, _ = model_ops._calls.layout(torch.zeros(6, 0, 16).transpose(0, 1))
    assert (rows, cols) == (0, 16)
    rows, cols, _, _ = model_ops._calls.layout(torch.zeros(0, 6).t())
    assert (rows, cols) == (6, 0)
    rows, cols, _, _ = model_ops._calls.layout(torch.zeros(6, 0).t())
    assert (rows, cols) == (0, 6)


@pytest.mark.parametrize("op,name", [("sort", "dest"), ("sort", "source"), ("sort", "offsets"),
                                     ("dispatch", "dest"), ("dispatch", "source"), ("combine", "dest"),
                                     ("combine_grad", "dest"), ("combine_grad", "source")])
def test_routing_is_aligned(dcopy, op, name):
    """An array that does not start on its elements' alignment is refused, not read."""
    places = places_of(dcopy, op)
    at, *rest = places[name]
    for off in (1, 2, 3):
        rc, message = call_at(dcopy, op, {**places, name: (at + off, *rest)})
        assert rc == dcopy.ERR_PARAM_INVALID and b"not aligned" in message and name.encode() in message


def test_numbers_are_aligned(dcopy):
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    lib, built = dcopy.lib(), dcopy.DcopyGradList()
    built.workspace = BASE
    ref, far = ctypes.byref(built), BASE + (1 << 20)
    for call in (lambda: lib.dcopy_grad_sum_squares(ref, far + 4, None),
                 lambda: lib.dcopy_grad_clip(ref, far + 4, 1.0, 0.0, None, None),
                 lambda: lib.dcopy_grad_clip(ref, far, 1.0, 0.0, far + 10, None),
                 lambda: lib.dcopy_clip_grad_norm(ref, 1.0, 0.0, far + 2, None)):
        assert call() == dcopy.ERR_PARAM_INVALID and b"not aligned" in lib.dcopy_last_error_message()


def test_first_ids_at_the_end_of_the_range(dcopy):
    """A part of a vocabulary whose ids would pass 2^63 is refused: ids from the other end of
    the range would fall into it."""
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    lib, m = dcopy.lib(), _mat(dcopy)
    ids, out = _mat(dcopy, 0x40000, 4, 1, 1, 9), _mat(dcopy, 0x20000)
    top = (1 << 63) - 1
    for first, refused in ((top, True), (top - 2, True), (top - 3, False), (-top - 1, False)):
        for rc in (lib.dcopy_embedding_lookup(out, m, ids, first, 1.0, None),
                   lib.dcopy_embedding_grad(m, out, ids, first, 1.0, 0, 0x80000, 1 << 20, None)):
            assert (rc == dcopy.ERR_PARAM_INVALID) == refused, (first, lib.dcopy_last_error_message())
