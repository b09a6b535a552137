"""The loss of a gradient-free forward with 8-bit layers and head, on a real MI355X."""
import pytest
import torch

from test_gpu_fp8_model import batch, make

pytestmark = pytest.mark.gpu


@torch.no_grad()
@pytest.mark.parametrize("fp32_residual", [False, True])
@pytest.mark.parametrize("kw", [dict(), dict(normalize_by="tokens"), dict(seq_weight=True)])
def test_loss_without_gradients_is_that_of_the_logits(dev, kw, fp32_residual):
    """masked_token_loss uses the 8-bit head where the forward does: the same loss as that of the forward's logits."""
    from src.loss import variational_lower_bound_loss
    tr = make(dev, fp8_head=True, fp32_residual=fp32_residual).eval().transformer
    for p in tr.output_layer.parameters():      # (logits of ordinary size, so that the heads differ by more than rounding)
        p.mul_(20.0)
    ids, att = batch(dev)
    g = torch.Generator().manual_seed(8)
    targets = torch.randint(104, 700, ids.shape, generator=g).to(dev)
    if "seq_weight" in kw:
        kw = dict(seq_weight=torch.tensor([1.0, 3.0, 0.5], device=dev))
    got = tr.masked_token_loss(ids, targets, 103, att, **kw)
    want = variational_lower_bound_loss(logits=tr(ids, att), targets=targets, masked_input_ids=ids, mask_token_id=103,
                                        attention_mask=att, **kw)
    tr.fp32_logits = True      # (the same values, widened)
    assert tr(ids, att).dtype == torch.float32
    assert abs(float(tr.masked_token_loss(ids, targets, 103, att, **kw)) - float(want)) <= 40 * 2.0 ** -24 * abs(float(want))
    # (fp32 sums of at most 40 masked rows' losses, all of one sign, maybe in another order)
    assert abs(float(got) - float(want)) <= 40 * 2.0 ** -24 * abs(float(want))
    tr.fp8_head = False
    other = tr.masked_token_loss(ids, targets, 103, att, **kw)
    assert abs(float(other) - float(want)) > 1e-5 * abs(float(want))
