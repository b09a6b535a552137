"""The 8-bit copies of weights: modes, threads, replaced parameters, on a real MI355X."""
import pytest
import torch

from test_gpu_fp8 import make_layer
from test_gpu_fp8_model import batch, make

pytestmark = pytest.mark.gpu


def test_copies_made_in_inference_mode_are_written_again_outside_it(dev):
    from src import ops
    lin, packs = make_layer(dev)
    x = torch.randn(5, 192, device=dev).bfloat16()
    with torch.inference_mode():
        y0 = ops.fp8_linear(x, packs[2])
    with torch.no_grad():
        lin[3].weight.mul_(2.0)
        lin[3].bias.mul_(2.0)
        assert torch.equal(ops.fp8_linear(x, packs[2]), 2 * y0)
        lin[3].weight.mul_(2.0)
        lin[3].bias.mul_(2.0)
    with torch.inference_mode():          # and the other way round
        assert torch.equal(ops.fp8_linear(x, packs[2]), 4 * y0)


def test_threads_with_streams_of_their_own(dev):
    import threading

    from src import ops
    lin, packs = make_layer(dev)
    x = torch.randn(300, 192, device=dev).bfloat16()
    with torch.no_grad():
        want = ops.fp8_linear(x, packs[2])
    for step in range(4):
        torch.cuda.synchronize()
        start, out, failed = threading.Barrier(4), [None] * 4, []

        def call(i):
            try:
                with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
                    start.wait()
                    out[i] = ops.fp8_linear(x, packs[2])
            except BaseException as e:
                failed.append(e)
        threads = [threading.Thread(target=call, args=(i,)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not failed, failed
        assert all(torch.equal(y, want) for y in out)
        with torch.no_grad():
            lin[3].weight.mul_(2.0)
            lin[3].bias.mul_(2.0)
        want = 2 * want


@torch.no_grad()
def test_parameters_replaced_by_others(dev):
    tr, other = make(dev, fp8_head=True).eval().transformer, make(dev, fp8_head=True).eval().transformer
    for p in other.parameters():
        p.add_(0.01 * torch.randn_like(p))
    ids, att = batch(dev)
    tr(ids, att)
    want = other(ids, att)
    tr.load_state_dict(other.state_dict(), assign=True)
    assert torch.equal(tr(ids, att), want)
