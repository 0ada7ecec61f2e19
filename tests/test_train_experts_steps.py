"""The expert example's steps do not wait for the device."""

import sys

import pytest
import torch

import adambridge_amd as ab
from test_train_experts import example


def test_losses_are_read_when_the_steps_are_done(monkeypatch):
    """On the CPU: the example makes no loss a Python number before the last step's update."""
    steps, reads = [], []
    step, item = torch.optim.AdamW.step, torch.Tensor.item

    def counted_step(self, *args):
        steps.append(0)
        return step(self, *args)

    def noted_item(self):
        if sys._getframe(1).f_code.co_filename == example.__file__:
            reads.append(len(steps))
        return item(self)

    monkeypatch.setattr(torch.optim.AdamW, "step", counted_step)
    monkeypatch.setattr(torch.Tensor, "item", noted_item)
    losses, _, _ = example.train(3, "cpu", "bf16", batch=2)
    assert len(losses) == len(steps) == 3 and reads == [3, 3, 3]


@pytest.mark.gpu
def test_a_step_has_no_synchronizing_call():
    torch.manual_seed(0)
    model = example.Model().to("cuda", torch.bfloat16)
    opt = ab.AdamBridge(model.parameters(), lr=3e-3, precision="bf16")
    ids = torch.randperm(512)[:16].repeat(6).cuda()
    example.fit(model, opt, ids, 2, 8, 64)   # builds the optimizer's state
    before = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        losses = example.fit(model, opt, ids, 3, 8, 64)
    finally:
        torch.cuda.set_sync_debug_mode(before)
    assert len(losses) == 3 and all(loss.is_cuda and loss.isfinite() for loss in losses)
    opt.close()
