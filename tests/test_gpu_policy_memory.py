"""GPU: what ``policy.lm_head_token_logps`` does where memory is short: the products that it may keep for the backward pass
are kept only if there is room for them."""

import pytest
import torch

from genrec_amd.policy import lm_head_token_logps

pytestmark = pytest.mark.gpu

N, H, V = 8192, 64, 80000  # 2.6 GB of products, 1 GB for a chunk of their gradient


def _step(hidden, weight, ids, g, **options):
    x, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    lp = lm_head_token_logps(x, w, ids, **options)
    held = torch.cuda.max_memory_allocated() - base
    return held, (lp.detach(), *torch.autograd.grad(lp, [x, w], g))


def test_products_are_kept_only_where_there_is_room():
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(1)
    hidden = torch.randn((N, H), generator=gen, device=dev).to(torch.bfloat16)
    weight = (torch.randn((V, H), generator=gen, device=dev) * 0.3).to(torch.bfloat16)
    ids = torch.randint(0, V, (N,), generator=gen, device=dev)
    g = torch.randn((N,), generator=gen, device=dev)
    lean, want = _step(hidden, weight, ids, g, keep_bytes=0)
    full, kept = _step(hidden, weight, ids, g)
    assert lean < N * V * 4 <= full
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(dev).total_memory
    try:  # the allocator refuses more than 2 GB on top of what is held
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (2 << 30)) / total, dev)
        held, got = _step(hidden, weight, ids, g)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0, dev)
    assert held < N * V * 4
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(_step(hidden, weight, ids, g)[1], kept))
