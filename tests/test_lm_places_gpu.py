"""Plans that a program made or changed itself."""
import pytest

torch = pytest.importorskip("torch")
from test_lm_gpu import DEV, TYPES, lm, rand  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("channels", [24, 1029])
def test_places_outside_the_rows_count_as_dropped(lm, dtype, channels):
    gen = torch.Generator().manual_seed(channels)
    T, K, E = 37, 3, 5
    plan = lm.route(torch.randint(0, E, (T, K), generator=gen, dtype=torch.int32).to(DEV), E)
    wild = torch.rand(T, K, generator=gen).to(DEV) < 0.3
    odd = torch.tensor([T * K, T * K + 1, 2 ** 31 - 1, -2, -2 ** 31], dtype=torch.int32, device=DEV)
    odd = odd[torch.randint(0, len(odd), (T, K), generator=gen).to(DEV)]
    dropped = lm.Route(plan.offsets, plan.order, torch.where(wild, -1, plan.place))
    outside = lm.Route(plan.offsets, plan.order, torch.where(wild, odd, plan.place))
    x, y, dout = (rand(gen, n, channels, dtype=dtype).to(DEV) for n in (T, T * K, T))
    w = torch.rand(T, K, generator=gen).to(DEV)
    live = dropped.place[dropped.place >= 0].long()
    assert torch.equal(lm.gather_tokens(x, outside)[live], lm.gather_tokens(x, dropped)[live])
    assert torch.equal(lm.combine_tokens(y, outside, w), lm.combine_tokens(y, dropped, w))
    assert torch.equal(lm.gather_tokens_backward(y, outside), lm.gather_tokens_backward(y, dropped))
    (dy, dw), (ey, ew) = lm.combine_tokens_backward(dout, y, outside, w), lm.combine_tokens_backward(dout, y, dropped, w)
    assert torch.equal(dy[live], ey[live]) and torch.equal(dw, ew) and (dw[wild] == 0).all()


def test_plans_of_other_types_are_refused(lm):
    place = torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    for bad in (place, place.int().flatten(), place.int().t()):
        with pytest.raises(ValueError):
            lm.Route(None, None, bad)
