"""GPU: tree_attention when a bounded wait inside it runs out.

A build of tree_attention.cu that checks itself (TABBY_CHECKS=1, waits of 2 ms) withholds a
sequence's value tiles, or lets a warp that issues products give up with one on its way. The
kernel has to return, what the wait concerns has to be NaN (withheld tiles: every slot in use of
the sequence), everything else equal to the ordinary build's outputs or, where the same CTA had it
still to do, NaN; no CTA may give its tensor memory back before its products are done; and the
next call has to be right. No GPU fault is involved: the waits give up.
"""
import ctypes

import pytest

from tests.conftest import gpu_available

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def checked(tmp_path_factory):
    if not gpu_available():
        pytest.skip("no CUDA device")
    from tabby_b200 import _lib, build

    try:
        build.nvcc()
    except RuntimeError:
        pytest.skip("no nvcc")
    path = str(tmp_path_factory.mktemp("checked") / "libtree.so")
    build._build_lib(path, ["decode_capi.cu", "tree_attention.cu"], False,
                     ("TABBY_CHECKS=1", "TABBY_WAIT_NS=2000000ull"))
    names = ("tabby_tree_workspace_bytes", "tabby_tree_attention_async",
             "tabby_decode_last_error")
    lib = _lib._load(path, {n: _lib.DECODE_SIGNATURES[n] for n in names})
    lib.tabby_debug_tree.argtypes = [ctypes.c_int32, ctypes.c_int32,
                                     ctypes.POINTER(ctypes.c_int32)]
    return lib


def attend(lib, q, k, v, lengths, parents):
    from tabby_b200 import _lib as m

    b, n, hq, d = q.shape
    hk, entries = k.shape[1:3]
    size = ctypes.c_size_t()
    assert lib.tabby_tree_workspace_bytes(b, n, hq, hk, d, ctypes.byref(size)) == 0
    work = torch.empty(size.value, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(q)
    a = m.TreeAttentionArgs()
    for name, x in (("q", q), ("k", k), ("v", v), ("out", out), ("lengths", lengths),
                    ("parents", parents), ("workspace", work)):
        setattr(a, name, x.data_ptr())
    for name, x, axes in (("q", q, ("batch", "node", "head")), ("k", k, ("batch", "head", "entry")),
                          ("v", v, ("batch", "head", "entry")),
                          ("out", out, ("batch", "node", "head"))):
        for i, axis in enumerate(axes):
            setattr(a, f"{name}_{axis}_stride", x.stride(i))
    a.parents_stride, a.dtype = parents.stride(0), m.TABBY_BF16
    a.batch, a.nodes, a.heads, a.kv_heads, a.dim, a.entries = b, n, hq, hk, d, entries
    a.scale, a.workspace_bytes = d ** -0.5, size.value
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.tabby_tree_attention_async(0, a, stream) == 0, lib.tabby_decode_last_error()
    torch.cuda.synchronize()
    return out


def debug(lib, withhold=-1, give_up=-1):
    n = ctypes.c_int32()
    assert lib.tabby_debug_tree(withhold, give_up, ctypes.byref(n)) == 0
    return n.value


# Workers with a tile each (the first), with several, with whole items; one and two row tiles.
@pytest.mark.parametrize("batch,nodes,heads,kv_heads,dim,length", [
    (3, 5, 2, 1, 64, 300), (6, 9, 8, 4, 64, 3000), (6, 26, 32, 8, 128, 1500),
    (40, 4, 16, 8, 64, 70), (5, 64, 8, 2, 80, 900),
])
@pytest.mark.parametrize("how", ["withhold", "give_up"])
def test_a_wait_that_runs_out(checked, batch, nodes, heads, kv_heads, dim, length, how):
    import tabby_b200 as tb

    g = torch.Generator(device="cuda").manual_seed(length)

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g).bfloat16()

    q = rand(batch, nodes, heads, dim)
    k, v = (rand(batch, kv_heads, length + nodes, dim) for _ in "kv")
    lengths = torch.full((batch,), length, dtype=torch.int32, device="cuda")
    parents = torch.tensor([[-1] + [(j - 1) // 2 for j in range(1, nodes)]] * batch,
                           dtype=torch.int32, device="cuda")
    want = tb.tree_attention(q, k, v, lengths, parents)
    debug(checked)
    assert torch.equal(attend(checked, q, k, v, lengths, parents), want)
    bad = batch // 2
    debug(checked, **{how: bad})
    got = attend(checked, q, k, v, lengths, parents)
    assert debug(checked) == 0  # CTAs with products on their way, and nothing withheld again
    nan = got.isnan()
    assert torch.equal(got[~nan], want[~nan])
    if how == "withhold":
        assert nan[bad].all()
        # A CTA takes one tile, or goes on from one sequence into the next at most.
        apart = {3: 0, 5: 1, 6: 1, 40: 2}[batch]
        assert not nan[[b for b in range(batch) if abs(b - bad) > apart]].any()
    assert torch.equal(attend(checked, q, k, v, lengths, parents), want)
