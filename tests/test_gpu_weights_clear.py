"""New keys' places among the weights of a cache in pages."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages,hkv,page,tokens", [(1, 1, 16, 1), (9, 3, 16, 50), (40, 8, 64, 1500), (5, 7, 1024, 4999), (300, 2, 32, 0)])
def test_new_places_are_zero_and_others_stay(gpu_device, pages, hkv, page, tokens):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(tokens)
    weights = torch.rand(pages, hkv, page, generator=gen)
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    for i, bad in enumerate((-1, pages * page, 1 << 40)):
        if tokens > 3:
            slots[7 * i + 1] = bad
    whole = torch.full((pages, hkv + 2, page + 3), 5.0)
    whole[:, 1:1 + hkv, :page] = weights
    want = whole.clone()
    for s in slots.tolist():
        if 0 <= s < pages * page:
            want[s // page, 1:1 + hkv, s % page] = 0
    dense, live = weights.to(gpu_device), whole.to(gpu_device)
    ops.paged_weights_clear(dense, slots.to(gpu_device))
    ops.paged_weights_clear(live[:, 1:1 + hkv, :page], slots.to(gpu_device))  # (rows and pages that do not follow each other)
    assert torch.equal(live.cpu(), want) and torch.equal(dense.cpu(), want[:, 1:1 + hkv, :page])
    with torch.cuda.stream(torch.cuda.Stream(gpu_device)) as _:
        again = weights.to(gpu_device)
        ops.paged_weights_clear(again, slots.to(gpu_device))
        torch.cuda.current_stream(gpu_device).synchronize()
    assert torch.equal(again, dense)


def test_refusals(gpu_device):
    from shareprefill_amd import ops

    weights, slots = torch.zeros(4, 2, 16, device=gpu_device), torch.zeros(3, dtype=torch.int64, device=gpu_device)
    for call in (lambda: ops.paged_weights_clear(weights.double(), slots), lambda: ops.paged_weights_clear(weights.transpose(1, 2), slots),
                 lambda: ops.paged_weights_clear(weights[0], slots), lambda: ops.paged_weights_clear(weights.cpu(), slots),
                 lambda: ops.paged_weights_clear(weights, slots.int()), lambda: ops.paged_weights_clear(weights, slots.cpu()),
                 lambda: ops.paged_weights_clear(weights, slots[None])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        ops.paged_weights_clear(torch.zeros(4, 2, 24, device=gpu_device), slots)
