"""KV4Cache's fields after construction: what is set takes effect with the next
call, what does not fit is refused and changes nothing."""
from __future__ import annotations

import copy
import dataclasses

import pytest
import torch

from rans_vectoradd import kv4


def filled(dev, seed, gains=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    arrays = [torch.randint(0, 256, (4, 2, 16, 64), device=dev, generator=g, dtype=torch.uint8),
              torch.randint(0x20, 0x40, (4, 2, 16, 8), device=dev, generator=g, dtype=torch.uint8)]
    arrays += [t.flip(0) for t in arrays]
    return kv4.KV4Cache(*arrays, *([torch.tensor([0.5, 3.0], device=dev), torch.tensor([7.0, 0.25], device=dev)] if gains else []))


def results(cache, dev):
    slots = torch.arange(64, device=dev)
    q = torch.ones(1, 4, 128, dtype=torch.bfloat16, device=dev)
    table, lens = torch.arange(4, dtype=torch.int32, device=dev)[None], torch.tensor([64], dtype=torch.int32, device=dev)
    return torch.cat([*(t.flatten() for t in kv4.read(cache, slots, torch.float32)), kv4.attention(cache, q, table, lens).flatten()])


@pytest.mark.gpu
@pytest.mark.parametrize("field", ["k_codes", "k_scales", "v_codes", "v_scales", "k_gain", "v_gain"])
def test_a_set_field_takes_effect(cuda, field):
    cache, other = filled(cuda, 1), filled(cuda, 2, gains=True)
    before, old = results(cache, cuda), getattr(cache, field)
    setattr(cache, field, getattr(other, field))
    got = results(cache, cuda)
    assert getattr(cache, field) is getattr(other, field)
    want = results(dataclasses.replace(filled(cuda, 1), **{field: getattr(other, field)}), cuda)
    assert torch.equal(got, want) and not torch.equal(got, before)
    setattr(cache, field, old)
    assert torch.equal(results(cache, cuda), before)


@pytest.mark.gpu
def test_append_goes_to_the_arrays_that_were_set(cuda):
    cache = filled(cuda, 3)
    old, new = cache.k_codes, torch.zeros_like(cache.k_codes)
    keep = old.clone()
    cache.k_codes = new
    x = torch.randn(3, 2, 128, device=cuda).to(torch.bfloat16)
    kv4.append(cache, x, x, torch.tensor([0, 17, 63], device=cuda))
    assert torch.equal(old, keep) and new.any()


@pytest.mark.gpu
def test_what_does_not_fit_is_refused_and_changes_nothing(cuda):
    cache = filled(cuda, 4, gains=True)
    before = results(cache, cuda)
    bigger = torch.zeros(8, 2, 16, 64, dtype=torch.uint8, device=cuda)
    for field, value in (("k_codes", bigger), ("k_codes", cache.k_codes.cpu()), ("v_scales", cache.v_scales.float()),
                         ("v_codes", bigger[::2]), ("k_gain", torch.ones(3, device=cuda)), ("v_gain", torch.ones(2)),
                         ("k_gain", torch.ones(2, device=cuda, dtype=torch.float64))):
        old = getattr(cache, field)
        with pytest.raises(RuntimeError):
            setattr(cache, field, value)
        assert getattr(cache, field) is old
    with pytest.raises(AttributeError):
        del cache.k_gain
    assert torch.equal(results(cache, cuda), before)
    cache.note = "what a caller keeps with it"
    assert cache.note


@pytest.mark.gpu
def test_copies_are_independent(cuda):
    cache = filled(cuda, 5)
    before, twin = results(cache, cuda), copy.copy(cache)
    twin.v_gain = torch.tensor([2.0, 4.0], device=cuda)
    assert cache.v_gain is None and torch.equal(results(cache, cuda), before)
    assert not torch.equal(results(twin, cuda), before)
