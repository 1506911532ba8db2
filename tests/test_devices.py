"""Calls on tensors of a device that is not the current one."""
import contextlib

import pytest
import torch

from strim_amd import ops


def test_a_call_runs_with_its_device_current(monkeypatch):
    """Without a GPU: the device that is made current, and none where it is already."""
    made = []

    @contextlib.contextmanager
    def device(d):
        made.append(d)
        yield

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    zero, one = torch.device("cuda:0"), torch.device("cuda:1")
    assert not ops._elsewhere(None, zero) and ops._elsewhere(None, one)
    assert ops._there(lambda *a: (a, list(made)), None, one, 1, 2) == ((1, 2), [one])


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_second_device():
    """The operators on the second device with the first one current, and after calls there: the same
    bits."""
    g = torch.Generator().manual_seed(1)
    h, w = torch.randn(6, 1024, generator=g).bfloat16(), torch.randn(900, 1024, generator=g).bfloat16()
    nw, t = torch.randn(1024, generator=g).bfloat16(), torch.randint(0, 900, (6,), generator=g).int()
    out = []
    for dev in ("cuda:0", "cuda:1"):
        a, b, n, ids = h.to(dev), w.to(dev), nw.to(dev), t.to(dev)
        q = ops.q4_pack(b, 64)
        loss, lse, _ = ops.head_loss(a, b, ids)
        res = [loss, *ops.head_loss_grad(a, b, ids, lse, lse), q.words, ops.q4_unpack(q),
               ops.head_logits_q4(a, q, n), ops.head_logits_q4(a.repeat(4, 1), q), ops.head_logits(a, b, n)]
        out.append([r.cpu() for r in res])
    assert torch.cuda.current_device() == 0
    for x, y in zip(*out):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_stream_of_another_device_is_refused():
    class Other(torch.cuda.Stream):
        device = torch.device("cuda:1")

    h, w = torch.zeros(1, 64, device="cuda:0").bfloat16(), torch.zeros(9, 64, device="cuda:0").bfloat16()
    with pytest.raises(ValueError, match="stream"):
        ops.head_loss(h, w, torch.zeros(1, dtype=torch.int32, device="cuda:0"), stream=Other())
