"""An error that other code left on the thread is neither reported as an operator's nor taken from whom it belongs to."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
from test_lm_gpu import DEV, lm, rand, random_pattern  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def test_errors_of_others_stay_theirs(lm):
    from nsparse_amd.capi import load_lm
    lib = load_lm()
    gen = torch.Generator().manual_seed(91)
    n, H, G, D, B, W = 2100, 4, 2, 64, 16, 4
    q, k, v, dout = (rand(gen, n, h, D, dtype=torch.bfloat16).to(DEV) for h in (H, G, G, H))
    idx = random_pattern(gen, n, G, W, 100).to(DEV)
    T, K, E, Ch = 5000, 2, 4, 8
    ids = torch.randint(0, E, (T, K), generator=gen, dtype=torch.int32).to(DEV)
    x, w = rand(gen, T, Ch).to(DEV), torch.rand(T, K, generator=gen).to(DEV)

    def bufs():
        e = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=DEV)
        return dict(means=e(-(-n // B), G, D), idx=e(n, G, W, t=torch.int32), out=e(n, H, D), lse=e(n, H, t=torch.float32), dq=e(n, H, D),
                    dk=e(n, G, D), dv=e(n, G, D), offsets=e(E + 1, t=torch.int32), order=e(T * K, t=torch.int32), place=e(T, K, t=torch.int32),
                    xs=e(T * K, Ch, t=torch.float32), y=e(T, Ch, t=torch.float32), dy=e(T * K, Ch, t=torch.float32), dw=e(T, K, t=torch.float32))

    a, _ = lm._attn(lm.Seqs(1), B, q=q, k=k, v=v, width=W, causal=True, scale=0.125, first=1, local=1)
    r = C.byref(a)
    need, need_route = lib.nsparse_lm_block_attention_bwd_workspace(r), lib.nsparse_lm_route_workspace(T, K, E)
    ws, ws_route = (torch.zeros(max(m, 16), dtype=torch.uint8, device=DEV) for m in (need, need_route))
    st = torch.cuda.current_stream().cuda_stream

    def calls(b):
        p = {name: t.data_ptr() for name, t in b.items()}
        yield lib.nsparse_lm_block_means(r, k.data_ptr(), p["means"], 0, st)
        yield lib.nsparse_lm_select_blocks(r, q.data_ptr(), p["means"], p["idx"], st)
        yield lib.nsparse_lm_block_attention(r, q.data_ptr(), k.data_ptr(), v.data_ptr(), idx.data_ptr(), p["out"], p["lse"], st)
        yield lib.nsparse_lm_block_attention_bwd(r, q.data_ptr(), k.data_ptr(), v.data_ptr(), idx.data_ptr(), p["out"], p["lse"],
                                                 dout.data_ptr(), p["dq"], p["dk"], p["dv"], ws.data_ptr(), need, st)
        yield lib.nsparse_lm_route(ids.data_ptr(), T, K, E, p["offsets"], p["order"], p["place"], ws_route.data_ptr(), need_route, st)
        yield lib.nsparse_lm_gather_tokens(0, x.data_ptr(), p["place"], T, K, Ch, p["xs"], st)
        yield lib.nsparse_lm_combine_tokens(0, p["xs"], p["place"], w.data_ptr(), T, K, Ch, p["y"], st)
        yield lib.nsparse_lm_combine_tokens_bwd(0, x.data_ptr(), p["xs"], p["place"], w.data_ptr(), T, K, Ch, p["dy"], p["dw"], st)

    want, got = bufs(), bufs()
    assert list(calls(want)) == [0] * 8
    torch.cuda.synchronize()
    left = lib.dll.hipSetDevice(9999)
    assert left != 0
    seen, last = list(calls(got)), lib.dll.hipGetLastError()  # reading it takes it away before torch looks
    assert seen == [0] * 8 and last == left
    assert all(torch.equal(want[name], got[name]) for name in want)
