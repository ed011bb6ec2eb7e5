"""Options of ops.rotate_heads are taken by their values, whatever holds them: looked at without a GPU, and with one."""
import math

import numpy as np
import pytest
import torch

from featgraph_amd.module import rotate

F32 = torch.float32


def sizes(frequencies=None, base=10000.0, sections=None, rotary_len=None, interleaved=False, eps=1e-6):
    shape = torch.Size((1, 3, 2, 32))
    return rotate._plan(F32, shape, shape, False, *rotate._options(base, frequencies, sections, rotary_len, interleaved, eps)).sizes


def test_values_and_not_what_holds_them():
    numbers = [0.5 ** i for i in range(16)]
    right = sizes(numbers)
    for held in (tuple(numbers), np.array(numbers), torch.tensor(numbers), torch.tensor(numbers, dtype=torch.float64), [torch.tensor(x) for x in numbers], list(np.float32(numbers))):
        assert sizes(held) == right
    assert sizes([1] * 16) == sizes([1.0] * 16) != right
    assert sizes(base=10000) == sizes(base=np.float32(10000)) == sizes(base=torch.tensor(10000.0)) == sizes()
    assert sizes(eps=torch.tensor(0.25)) == sizes(eps=0.25) != sizes()
    assert sizes(sections=torch.tensor([4, 12])) == sizes(sections=(4, 12)) == sizes(sections=[np.int64(4), torch.tensor(12)])
    assert sizes(rotary_len=torch.tensor(16)) == sizes(rotary_len=16) and sizes(interleaved=1) == sizes(interleaved=True)


def test_numbers_that_change_where_they_are():
    held, base, parts = [torch.tensor(1.0) for _ in range(16)], torch.tensor(10000.0), [torch.tensor(16), torch.tensor(0)]
    first = sizes(held), sizes(base=base), sizes(sections=parts)
    for x in held:
        x.mul_(0.5)
    base.mul_(2)
    parts[0].sub_(4), parts[1].add_(4)
    assert sizes(held) == sizes([0.5] * 16) != first[0] and sizes(base=base) == sizes(base=20000.0) != first[1]
    assert sizes(sections=parts) == sizes(sections=(12, 4)) != first[2]


def test_a_tensor_is_looked_up():
    buffer = torch.rand(16)
    sizes(buffer)
    before = rotate._plan.cache_info()
    for _ in range(5):
        sizes(buffer)
    after = rotate._plan.cache_info()
    assert after.hits == before.hits + 5 and after.currsize == before.currsize


def test_what_is_no_number():
    for bad in (dict(sections=(16.0, 0.0)), dict(sections=[torch.tensor(16.0)]), dict(rotary_len=16.0), dict(frequencies=torch.ones((4, 4)))):
        sizes(sections=(16, 0)), sizes(rotary_len=16), sizes([1.0] * 16)        # equal ones are kept
        with pytest.raises(TypeError):
            sizes(**bad)
    for bad in (dict(frequencies=[math.inf] * 16), dict(frequencies=torch.ones(15)), dict(base=torch.tensor(-1.0)), dict(eps=math.nan), dict(sections=(16, 1))):
        with pytest.raises(ValueError):
            sizes(**bad)


def test_learned_frequencies_are_refused():
    leaf = torch.ones(16, requires_grad=True)
    for bad in (dict(frequencies=leaf), dict(frequencies=list(leaf)), dict(base=leaf[0] * 2)):
        with pytest.raises(NotImplementedError, match="no gradient"):
            sizes(**bad)
    with torch.no_grad():
        assert sizes(leaf) == sizes([1.0] * 16)


@pytest.mark.gpu
def test_tensors_on_the_gpu():
    from featgraph_amd import ops
    q = torch.randn((2, 9, 4, 64), device="cuda")
    buffer = 10000.0 ** (-torch.arange(32, device="cuda", dtype=torch.float64) / 32)
    right = ops.rotate_heads(q, q, frequencies=buffer.tolist())[0]
    assert torch.equal(ops.rotate_heads(q, q, frequencies=buffer)[0], right)
    held = list(buffer.cpu())
    ops.rotate_heads(q, q, frequencies=held)
    for x in held:
        x.mul_(0.5)
    assert torch.equal(ops.rotate_heads(q, q, frequencies=held)[0], ops.rotate_heads(q, q, frequencies=(buffer / 2).tolist())[0])
    graph = torch.cuda.CUDAGraph()
    numbers = buffer.tolist()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="during capture"):
            ops.rotate_heads(q, q, frequencies=buffer)
        out = ops.rotate_heads(q, q, frequencies=numbers)[0]
    for _ in range(3):
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.rotate_heads(q, q, frequencies=numbers)[0])
