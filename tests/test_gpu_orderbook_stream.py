"""The order-book model served tick by tick over a paged cache: every step returns what the whole forward returns for
the ticks seen so far."""
import pytest
import torch

from ma_transformer_b200 import _native as nat
from ma_transformer_b200.layers.orderbook_model import OrderBookStream, OrderBookTransformer, synthetic_ticks
from helpers import orderbook_reference_forward as reference_forward

pytestmark = pytest.mark.gpu


def scaled(batch, n):
    t = synthetic_ticks(batch, n, seed=3)
    return (t - t.mean(dim=(0, 1))) / (t.std(dim=(0, 1)) + 1e-6)


@pytest.mark.parametrize("history", [0, 1, 131])
def test_steps_match_the_whole_forward(history):
    # the bars of the whole forward's own test: fp32 2e-3, bf16 0.08 of the logits' scale
    torch.manual_seed(0)
    model = OrderBookTransformer(taps=16, n_layers=2).eval()
    ticks = scaled(2, 150)
    with torch.no_grad():
        want = {n: reference_forward(model, ticks[:, :n]) for n in (history + 1, history + 9, 150)}
        for dtype, bar in ((torch.float32, 2e-3), (torch.bfloat16, 0.08)):
            model = model.cuda().to(dtype)
            t = ticks.cuda().to(dtype)
            stream = OrderBookStream(model, 2, 150, page_size=16)
            if history:
                first = stream.prefill(t[:, :history])
                ref = reference_forward(model.float().cpu(), ticks[:, :history])
                assert (first.float().cpu() - ref).abs().max() <= bar * max(1.0, float(ref.abs().max()))
                model.cuda().to(dtype)
            for n in range(history + 1, 151):
                got = stream.step(t[:, n - 1])
                if n in want:
                    assert (got.float().cpu() - want[n]).abs().max() <= bar * max(1.0, float(want[n].abs().max())), (dtype, n)
            assert nat.device_status() == 0
            with pytest.raises(ValueError, match="at most"):
                stream.step(t[:, 0])


def test_stream_refusals():
    stream = OrderBookStream(OrderBookTransformer(n_layers=1).cuda(), 2, 8)
    with pytest.raises(ValueError):
        stream.step(torch.zeros(3, 40, device="cuda"))
    with pytest.raises(ValueError):
        stream.prefill(torch.zeros(2, 9, 40, device="cuda"))
    stream.step(torch.zeros(2, 40, device="cuda"))
    with pytest.raises(ValueError, match="before the first"):
        stream.prefill(torch.zeros(2, 2, 40, device="cuda"))
    with pytest.raises(ValueError):
        OrderBookStream(OrderBookTransformer(n_layers=1).cuda(), 0, 8)
