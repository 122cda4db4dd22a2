"""Sequences whose arrays contradict themselves: nothing depends on what a workspace held, nothing beside the outputs is written."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
from test_lm_gpu import DEV, i32, lm, rand  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cu_q", [[0, 100, 50, 300], [0, 300, 150, 300], [0, 300, 10], [0, 10, 300], [300, 0, 300], [-7, 400, 120]], ids=str)
def test_gradient_of_rows_that_do_not_ascend(lm, cu_q):
    from nsparse_amd.capi import load_lm
    lib = load_lm()
    gen = torch.Generator().manual_seed(71)
    n, H, G, D, B, W, pad = 300, 4, 2, 64, 16, 4, 4096
    q, dout = (rand(gen, n, H, D, dtype=torch.bfloat16).to(DEV) for _ in range(2))
    k, v = (rand(gen, n, G, D, dtype=torch.bfloat16).to(DEV) for _ in range(2))
    idx = torch.zeros(n, G, W, dtype=torch.int32)
    idx[:, :, 1:] = torch.sort(torch.randint(1, 19, (n, G, W - 1), generator=gen, dtype=torch.int32), dim=2).values
    idx = idx.to(DEV)
    # every sequence has all keys to itself or none: gradients of key rows belong to one of them
    m = len(cu_q) - 1
    seqs = lm.Seqs(m, cu_q=i32(cu_q).to(DEV), cu_k=i32([0] + [n] * m).to(DEV))
    out, lse = lm.block_attention(q, k, v, idx, block=B, causal=False, seqs=seqs, return_lse=True)
    a, _ = lm._attn(seqs, B, q=q, k=k, v=v, width=W, causal=False, scale=0.125)
    need = lib.nsparse_lm_block_attention_bwd_workspace(C.byref(a))
    assert need > 0
    got = []
    for byte in (0, 255):
        room = [torch.full((t.numel() + 2 * pad,), 7.0, dtype=torch.bfloat16, device=DEV) for t in (q, k, v)]
        ws = torch.full((need,), byte, dtype=torch.uint8, device=DEV)
        assert lib.nsparse_lm_block_attention_bwd(C.byref(a), q.data_ptr(), k.data_ptr(), v.data_ptr(), idx.data_ptr(), out.data_ptr(),
                                                  lse.data_ptr(), dout.data_ptr(), *[r[pad:].data_ptr() for r in room], ws.data_ptr(), need,
                                                  torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert all((r[:pad] == 7).all() and (r[-pad:] == 7).all() for r in room)
        got.append(room)
    assert all(torch.equal(x, y) for x, y in zip(*got))
