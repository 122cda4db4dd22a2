"""libnsparse_lm.so without a GPU: exports, provenance, the layout of its argument block, refusals, and the oracle's own gradient."""
import ctypes as C
import glob
import hashlib
import os
import re
import subprocess

import pytest

import nsparse_amd as ns
from conftest import ROOT

torch = pytest.importorskip("torch")
import lm_oracle as lo  # noqa: E402

HEADER = os.path.join(ROOT, "include", "nsparse_lm.h")


@pytest.fixture(scope="module")
def lib():
    return ns.load_lm()


def test_exports_every_declared_symbol(lib):
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"^[A-Za-z_][\w \*]*?\b(\w+)\s*\([^;{]*\)\s*;", src, flags=re.M)))
    assert names == sorted(ns.LM_SIGNATURES)
    for n in names:
        assert hasattr(lib.dll, n)


def test_library_was_built_from_these_sources(lib):
    h = hashlib.sha256(open(HEADER, "rb").read())
    csrc = os.path.join(ROOT, "nsparse_amd", "csrc")
    for f in sorted(glob.glob(os.path.join(csrc, "lm", "*")), key=lambda p: os.path.relpath(p, csrc)):
        h.update(open(f, "rb").read())
    assert lib.nsparse_lm_build_info().decode() == "gfx950 " + h.hexdigest()[:16]


def test_argument_block_layout(tmp_path):
    fields = [f[0] for f in ns.LmAttn._fields_]
    prog = ["#include <stdio.h>", "#include <stddef.h>", '#include "nsparse_lm.h"', "int main(void){",
            'printf("size %zu\\n", sizeof(nsparse_lm_attn));']
    prog += [f'printf("{f} %zu\\n", offsetof(nsparse_lm_attn, {f}));' for f in fields] + ["return 0;}"]
    (tmp_path / "a.c").write_text("\n".join(prog))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "a.c"), "-o", str(tmp_path / "a")])
    got = dict(x.split() for x in subprocess.check_output([str(tmp_path / "a")], text=True).splitlines())
    assert int(got["size"]) == C.sizeof(ns.LmAttn)
    for f in fields:
        assert int(got[f]) == getattr(ns.LmAttn, f).offset, f


def _good(**change):
    a = ns.LmAttn()
    a.dtype, a.heads, a.kv_heads, a.head_dim, a.block, a.width, a.causal, a.n_seq = 2, 8, 2, 64, 16, 4, 1, 1
    a.q_rows = a.k_rows = 32
    a.q_stride[0], a.q_stride[1] = 512, 64
    for s in (a.k_stride, a.v_stride):
        s[1], s[2] = 128, 64
    for n, x in change.items():
        if isinstance(x, tuple):
            getattr(a, n)[x[0]] = x[1]
        else:
            setattr(a, n, x)
    return a


P = 4096  # an aligned address that no call below gets to read


@pytest.mark.parametrize("change, code", [
    (dict(dtype=3), -2), (dict(dtype=-1), -2), (dict(heads=0), -1), (dict(heads=9), -1), (dict(kv_heads=0), -1), (dict(head_dim=0), -1),
    (dict(head_dim=60), -1), (dict(head_dim=264), -1), (dict(block=8), -1), (dict(block=48), -1), (dict(block=512), -1), (dict(width=0), -1),
    (dict(width=257), -1), (dict(n_seq=0), -1), (dict(n_seq=3), -1), (dict(q_rows=-1), -1), (dict(k_rows=-1), -1), (dict(k_rows=2 ** 32), -1),
    (dict(q_rows=2 ** 31), -1), (dict(page_size=24), -1), (dict(page_size=16), -1), (dict(page_size=16, k_len=P), -1),
    (dict(page_size=16, k_len=P, page_table=P, cu_k=P), -1), (dict(page_size=16, k_len=P, page_table=P, table_stride=2 ** 40), -1),
    (dict(page_table=P), -1), (dict(q_stride=(0, 511)), -3), (dict(q_stride=(1, -64)), -3), (dict(k_stride=(1, 4)), -3),
    (dict(v_stride=(2, 63)), -3), (dict(page_size=16, k_len=P, page_table=P, table_stride=2, k_stride=(0, 1)), -3),
])
def test_refused_geometry(lib, change, code):
    a = _good(**change)
    assert lib.nsparse_lm_block_attention(C.byref(a), P, P, P, P, P, P, None) == code
    assert lib.nsparse_lm_last_error() == code and lib.nsparse_lm_last_error_string()


def test_refused_pointers_and_workspace(lib):
    a = _good()
    ref = C.byref(a)
    for bad in range(5):
        args = [P] * 5
        args[bad] = None
        assert lib.nsparse_lm_block_attention(ref, *args, None, None) == -1
    assert lib.nsparse_lm_block_attention(None, P, P, P, P, P, P, None) == -1
    assert lib.nsparse_lm_block_attention(ref, P + 2, P, P, P, P, P, None) == -3
    need = lib.nsparse_lm_block_attention_bwd_workspace(ref)
    assert need > 0
    assert lib.nsparse_lm_block_attention_bwd(ref, *[P] * 10, None, need, None) == -4
    assert lib.nsparse_lm_block_attention_bwd(ref, *[P] * 11, need - 1, None) == -4
    for bad in range(10):
        args = [P] * 11
        args[bad] = None
        assert lib.nsparse_lm_block_attention_bwd(ref, *args, need, None) == -1
    paged = _good(page_size=16, k_len=P, page_table=P, table_stride=2)
    assert lib.nsparse_lm_block_attention_bwd_workspace(C.byref(paged)) == -1
    assert lib.nsparse_lm_block_attention_bwd(C.byref(paged), *[P] * 11, need, None) == -1


def test_refused_selection(lib):
    for change in (dict(first=-1, local=1), dict(first=4, local=1), dict(local=0), dict(local=5), dict(causal=0, local=1), dict(first=2 ** 31 - 1, local=1)):
        a = _good(**change)
        assert lib.nsparse_lm_select_blocks(C.byref(a), P, P, P, None) == -1, change
    a = _good(local=1)
    for args in ((None, P, P), (P, None, P), (P, P, None)):
        assert lib.nsparse_lm_select_blocks(C.byref(a), *args, None) == -1
    assert lib.nsparse_lm_select_blocks(C.byref(a), P, P + 8, P, None) == -3
    assert lib.nsparse_lm_block_means(C.byref(a), None, P, 0, None) == -1
    assert lib.nsparse_lm_block_means(C.byref(a), P, P, -1, None) == -1
    assert lib.nsparse_lm_block_means(C.byref(a), P + 4, P, 0, None) == -3


def test_refused_routing(lib):
    assert lib.nsparse_lm_route_workspace(-1, 2, 8) == -1
    assert lib.nsparse_lm_route_workspace(4, 0, 8) == -1
    assert lib.nsparse_lm_route_workspace(4, 2, 0) == -1
    assert lib.nsparse_lm_route_workspace(4, 2, 4097) == -1
    assert lib.nsparse_lm_route_workspace(2 ** 30, 2, 8) == -1
    need = lib.nsparse_lm_route_workspace(100000, 2, 8)
    assert need > 0
    assert lib.nsparse_lm_route(P, 100000, 2, 8, P, P, P, None, need, None) == -4
    assert lib.nsparse_lm_route(P, 100000, 2, 8, P, P, P, P, need - 1, None) == -4
    assert lib.nsparse_lm_route(P, 100000, 2, 8, None, P, P, P, need, None) == -1
    assert lib.nsparse_lm_route(None, 100000, 2, 8, P, P, P, P, need, None) == -1
    assert lib.nsparse_lm_gather_tokens(3, P, P, 4, 2, 8, P, None) == -2
    assert lib.nsparse_lm_gather_tokens(0, P, P, 4, 0, 8, P, None) == -1
    assert lib.nsparse_lm_gather_tokens(0, P, None, 4, 2, 8, P, None) == -1
    assert lib.nsparse_lm_combine_tokens(0, P, P, P, 4, 2, 0, P, None) == -1
    assert lib.nsparse_lm_combine_tokens(0, P, P, P, 2 ** 31, 2, 8, P, None) == -1
    assert lib.nsparse_lm_combine_tokens(0, None, P, P, 4, 2, 8, P, None) == -1
    assert lib.nsparse_lm_combine_tokens_bwd(0, P, None, P, P, 4, 2, 8, P, P, None) == -1
    assert lib.nsparse_lm_combine_tokens_bwd(0, P, P, P, P, 4, 2, 8, P, None, None) == -1


def test_sizes_of_means_and_workspaces(lib):
    rows = lambda **c: lib.nsparse_lm_mean_rows(C.byref(_good(**c)))
    assert rows() == 2 and rows(k_rows=33) == 3 and rows(k_rows=0) == 0
    assert rows(n_seq=2) == 2 and rows(n_seq=2, k_rows=34) == 4
    assert rows(cu_k=P, n_seq=3, q_rows=33) == 5
    assert rows(page_size=32, k_len=P, page_table=P, table_stride=2, k_rows=7) == 14
    assert lib.nsparse_lm_route_workspace(512, 8, 1024) == 0  # one chunk needs none


def test_tensors_on_the_cpu_are_refused():
    from nsparse_amd import lm
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        lm.block_means(x, block=16)
    with pytest.raises(ValueError):
        lm.route(torch.zeros(4, 2, dtype=torch.int32), 4)
    with pytest.raises(ValueError):
        lm.Seqs(0)
    with pytest.raises(ValueError):
        lm.Seqs(2, cu_q=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError):
        lm.Seqs(2, k_len=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        lm.Seqs(2, page_table=torch.zeros(2, 4, dtype=torch.int32).t()[:2])


def test_oracle_gradient_against_differences():
    """The oracle's gradient formulas against central differences of its own forward."""
    gen = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    lay = lo.packed([5, 3], [9, 3])
    q, k, v, dout = r(8, 4, 8), r(12, 2, 8), r(12, 2, 8), r(8, 4, 8)
    idx = torch.tensor([[[0, 1, -1], [2, 1, 2]], [[0, 0, 2], [-1, -1, -1]]] * 4, dtype=torch.int32)
    f = lambda a, b, c: (lo.attention(a, b, c, idx, lay, 4, 0.3, True)["out"] * dout).sum()
    got = lo.attention(q, k, v, idx, lay, 4, 0.3, True, dout)
    for i, name in enumerate(("dq", "dk", "dv")):
        x = [q, k, v]
        step = r(*x[i].shape)
        h = 1e-5
        up, dn = list(x), list(x)
        up[i], dn[i] = x[i] + h * step, x[i] - h * step
        diff = (f(*up) - f(*dn)) / (2 * h)
        want = (got[name] * step).sum()
        assert abs(diff - want) < 1e-7 * (1 + abs(want)), name
