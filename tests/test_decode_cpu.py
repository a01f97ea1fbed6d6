"""CPU: libtabbydecode.so loads, exports exactly what include/tabby_decode.h declares, keeps
the struct layouts of the header, and refuses bad arguments before it touches a device."""
import ctypes
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "tabby_decode.h")
P = ctypes.c_void_p(4096)  # a pointer that is never followed


def _lib():
    from tabby_b200 import _lib as m

    return m, m.decode_lib()


def declared_symbols():
    return sorted(set(re.findall(r"TABBY_API\s+[\w\s\*]+?\b(tabby_\w+)\s*\(",
                                 open(HEADER).read())))


def test_library_exports_what_the_header_declares():
    m, L = _lib()
    names = declared_symbols()
    assert names == sorted(m.DECODE_SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", m.DECODE_LIB_PATH], capture_output=True,
                         text=True, check=True).stdout
    assert set(re.findall(r"\bT (tabby_\w+)", out)) == set(names)
    assert L.tabby_decode_abi_version() == 1


def test_struct_layouts_match_the_header(tmp_path):
    m, _ = _lib()
    src = tmp_path / "s.c"
    fields = [f for f, _ in m.TreeAttentionArgs._fields_]
    lay = [f for f, _ in m.StateLayout._fields_]
    src.write_text(
        '#include "tabby_decode.h"\n#include <stdio.h>\nint main(void) {\n'
        + "".join(f'printf("%zu\\n", offsetof(tabby_tree_attention_args, {f}));\n' for f in fields)
        + "".join(f'printf("%zu\\n", offsetof(tabby_state_layout, {f}));\n' for f in lay)
        + 'printf("%zu %zu\\n", sizeof(tabby_tree_attention_args), sizeof(tabby_state_layout));'
        + "return 0; }\n")
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"),
                    str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    want = [getattr(m.TreeAttentionArgs, f).offset for f in fields]
    want += [getattr(m.StateLayout, f).offset for f in lay]
    want += [ctypes.sizeof(m.TreeAttentionArgs), ctypes.sizeof(m.StateLayout)]
    assert [int(x) for x in got] == want


def _beam(L, **kw):
    a = dict(device=0, logits=P, dtype=0, batch_stride=400, beam_stride=100, batch=2, beams=4,
             vocab=100, scores=P, finished=None, eos=-1, n_out=8, next_scores=P, parents=P,
             tokens=P, next_finished=None, status=P, work=P, work_bytes=1 << 30, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return L.tabby_beam_step_async(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(batch=-1), b"batch"), (dict(beams=0), b"beams"), (dict(beams=65), b"beams"),
    (dict(vocab=0), b"vocab"), (dict(vocab=(1 << 30) + 1), b"vocab"),
    (dict(n_out=0), b"n_out"), (dict(n_out=129), b"n_out"), (dict(dtype=3), b"dtype"),
    (dict(eos=100), b"eos"), (dict(eos=-2), b"eos"), (dict(finished=P), b"eos"),
    (dict(batch_stride=-1), b"strides"), (dict(beam_stride=-1), b"strides"),
    (dict(logits=None), b"NULL"), (dict(scores=None), b"NULL"), (dict(status=None), b"NULL"),
    (dict(parents=None), b"NULL"), (dict(tokens=None), b"NULL"),
    (dict(next_scores=None), b"NULL"), (dict(logits=ctypes.c_void_p(4097)), b"aligned"),
    (dict(logits=ctypes.c_void_p(4098)), b"aligned"), (dict(work=None), b"workspace"),
    (dict(work_bytes=8), b"workspace"), (dict(work=ctypes.c_void_p(4104)), b"workspace"),
])
def test_beam_step_refuses(kw, text):
    m, L = _lib()
    assert _beam(L, **kw) == m.TABBY_EINVAL
    assert b"beam_step" in L.tabby_decode_last_error() and text in L.tabby_decode_last_error()


def test_empty_batches_do_nothing():
    m, L = _lib()
    assert _beam(L, batch=0, logits=None, work=None) == m.TABBY_OK
    lay = m.StateLayout(0, 0, 0, 4, 1, 1)
    assert L.tabby_states_reorder_async(0, None, 0, lay, 1, 1, P, None, None) == m.TABBY_OK
    assert L.tabby_states_reorder_async(0, None, 1, lay, 0, 1, P, None, None) == m.TABBY_OK
    assert L.tabby_tree_accept_async(0, P, 1, 1, P, P, 1, 0, 1, P, P, P, P, P, None, 0, None,
                                     None) == m.TABBY_OK


def _layout(m, row=1024, seg=256, ent=64, size=64, segments=4, entries=4):
    return m.StateLayout(row, seg, ent, size, segments, entries)


@pytest.mark.parametrize("lay,text", [
    (dict(segments=0), b"must be >= 1"), (dict(entries=0), b"must be >= 1"),
    (dict(size=0), b"must be >= 1"), (dict(size=1 << 31), b"2^31"), (dict(row=-1), b"strides"),
    (dict(seg=-1), b"strides"), (dict(ent=-1), b"strides"), (dict(row=0), b"overlap"),
    (dict(row=1023), b"overlap"), (dict(seg=255), b"overlap"), (dict(ent=63), b"overlap"),
    (dict(ent=0), b"overlap"),
])
def test_layouts_that_cannot_be_moved_in_place(lay, text):
    m, L = _lib()
    states = (ctypes.c_void_p * 1)(4096)
    assert L.tabby_states_reorder_async(0, states, 1, _layout(m, **lay), 2, 2, P, None,
                                        None) == m.TABBY_EINVAL
    assert text in L.tabby_decode_last_error()
    assert L.tabby_tree_accept_async(0, P, 1, 1, P, P, 1, 2, 1, P, P, P, P, P, states, 1,
                                     _layout(m, **lay), None) == m.TABBY_EINVAL
    assert text in L.tabby_decode_last_error() and b"accept" in L.tabby_decode_last_error()


def test_states_reorder_refuses():
    m, L = _lib()
    states = (ctypes.c_void_p * 2)(4096, None)
    lay = _layout(m)

    def call(states=states, n=2, lay=lay, batch=2, beams=2, parents=P):
        return L.tabby_states_reorder_async(0, states, n, lay, batch, beams, parents, None, None)

    for kw in (dict(n=-1), dict(batch=-1), dict(beams=0), dict(beams=65), dict(states=None),
               dict(parents=None), dict(lay=None), dict()):
        assert call(**kw) == m.TABBY_EINVAL, kw
    assert b"state 1 is NULL" in L.tabby_decode_last_error()


def test_states_reorder_checks_without_states():
    """What a call with states would refuse: the layout, and blocks past a launch's 2^31."""
    m, L = _lib()

    def call(lay, batch=2):
        return L.tabby_states_reorder_async(0, None, 0, lay, batch, 2, P, None, None)

    assert call(_layout(m)) == m.TABBY_OK
    assert call(_layout(m, row=0)) == m.TABBY_EINVAL
    assert b"overlap" in L.tabby_decode_last_error()
    many = (1 << 31) - 1
    assert call(_layout(m, row=many * 4, seg=4, ent=4, size=2, segments=many, entries=1)) \
        == m.TABBY_EINVAL
    assert b"too large" in L.tabby_decode_last_error()
    assert call(_layout(m, row=many * 4, seg=4, ent=4, size=2, segments=many, entries=1), 1) \
        == m.TABBY_OK


def test_tree_accept_refuses():
    m, L = _lib()
    caches = (ctypes.c_void_p * 1)(None)
    names = ("device", "sampled", "sb", "ss", "tokens", "parents", "ps", "batch", "nodes",
             "lengths", "path", "counts", "next", "next_lengths", "caches", "n", "lay", "stream")
    good = (0, P, 4, 1, P, P, 4, 2, 4, P, P, P, P, P, None, 0, None, None)
    for kw in (dict(batch=-1), dict(nodes=0), dict(nodes=65), dict(sb=-1), dict(ss=-1),
               dict(ps=-1), dict(sampled=None), dict(tokens=None), dict(parents=None),
               dict(lengths=None), dict(path=None), dict(counts=None), dict(next=None),
               dict(next_lengths=None), dict(n=-1), dict(n=1), dict(n=1, lay=_layout(m)),
               dict(n=1, lay=_layout(m), caches=caches)):
        a = dict(zip(names, good))
        a.update(kw)
        assert L.tabby_tree_accept_async(*a.values()) == m.TABBY_EINVAL, kw
        assert b"tree_accept" in L.tabby_decode_last_error()


def _tree_args(m, **kw):
    a = m.TreeAttentionArgs()
    good = dict(q=4096, k=4096, v=4096, out=4096, lengths=4096, parents=4096, parents_stride=4,
                dtype=m.TABBY_BF16, batch=2, nodes=4, heads=4, kv_heads=2, dim=64, entries=100,
                scale=0.125, workspace=4096, workspace_bytes=1 << 40, q_batch_stride=1024,
                q_node_stride=256, q_head_stride=64, k_batch_stride=12800, k_head_stride=6400,
                k_entry_stride=64, v_batch_stride=12800, v_head_stride=6400, v_entry_stride=64,
                out_batch_stride=1024, out_node_stride=256, out_head_stride=64)
    good.update(kw)
    for k, v in good.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(batch=-1), dict(nodes=0), dict(nodes=65), dict(heads=3), dict(kv_heads=0),
    dict(heads=0), dict(dim=0), dict(dim=4), dict(dim=60), dict(dim=136), dict(dtype=0),
    dict(dtype=7), dict(entries=0), dict(q=None), dict(k=None), dict(v=None), dict(out=None),
    dict(lengths=None), dict(parents=None), dict(q=4104), dict(k=4098), dict(v=4104),
    dict(out=4104), dict(k_entry_stride=60), dict(q_head_stride=-8), dict(parents_stride=-1),
    dict(workspace=None), dict(workspace=4104), dict(workspace_bytes=0),
    dict(scale=float("nan")), dict(scale=float("inf")),
])
def test_tree_attention_refuses(kw):
    m, L = _lib()
    assert L.tabby_tree_attention_async(0, _tree_args(m, **kw), None) == m.TABBY_EINVAL
    assert b"tree_attention" in L.tabby_decode_last_error()
    assert L.tabby_tree_attention_async(0, None, None) == m.TABBY_EINVAL


def test_no_device_is_an_error_not_an_abort():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    m, L = _lib()
    assert _beam(L) == m.TABBY_ECUDA
    assert L.tabby_tree_attention_async(0, _tree_args(m), None) == m.TABBY_ECUDA


def test_python_refuses_what_is_not_on_a_gpu():
    import torch

    import tabby_b200 as tb

    with pytest.raises(ValueError):
        tb.beam_step(torch.zeros(1, 2, 8), torch.zeros(1, 2))
    with pytest.raises(ValueError):
        tb.reorder_states([torch.zeros(2, 3)], torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(ValueError):
        z = torch.zeros(1, 4, dtype=torch.int32)
        tb.tree_accept(z, z, z, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(AttributeError):
        tb.no_such_operator


@pytest.mark.parametrize("shape,stride,with_entries,want", [
    # [rows, heads, entries, dim] bf16, head-major and token-major
    ((4, 2, 9, 64), (1152, 576, 64, 1), True, (2304, 1152, 128, 128, 2, 9)),
    ((4, 2, 9, 64), (1152, 64, 128, 1), True, (2304, 128, 256, 128, 2, 9)),
    # a state's own axes merge where memory allows
    ((4, 7, 3), (21, 3, 1), False, (42, 0, 0, 42, 1, 1)),
    ((4, 7, 3), (100, 10, 1), False, (200, 0, 20, 6, 1, 7)),
    ((4,), (1,), False, (2, 0, 0, 2, 1, 1)),
    ((1, 5), (0, 1), False, (0, 0, 0, 10, 1, 1)),
    ((4, 5, 6), (1, 24, 4), False, (2, 0, 8, 2, 1, 30)),
])
def test_state_layouts(shape, stride, with_entries, want):
    from tabby_b200.decode import _layout

    l = _layout(shape, stride, 2, with_entries)
    got = (l.row_stride, l.segment_stride, l.entry_stride, l.entry_bytes, l.segments, l.entries)
    assert got == want


def test_state_layouts_that_do_not_fit():
    from tabby_b200.decode import _layout

    with pytest.raises(ValueError):
        _layout((4, 9, 64), (576, 64, 1), 2, True)
    with pytest.raises(ValueError):
        _layout((4, 2, 9, 64), (1152, 576, 1, 9), 2, True)
    with pytest.raises(ValueError):
        _layout((4, 3, 4, 5, 6), (10000, 2000, 300, 40, 2), 2, False)
