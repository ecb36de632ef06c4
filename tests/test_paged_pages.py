"""Pages of DevicePagedKVBuffer that a window has left behind, and sequences that
go back."""
import pytest
import torch

from sbq.state import DevicePagedKVBuffer


def _held(b, i):
    return [j for j, id_ in enumerate(b.table[i].tolist()) if id_ >= 0]


def test_pages_behind_a_released_one():
    """A page that reserve does not give is an exception, never a token lost in silence."""
    b = DevicePagedKVBuffer(2, 2, 24, 12, 16, max_pages=6, device="cpu")
    b.reserve(0, 80)
    b.reserve(1, 20)
    b.length.copy_(torch.tensor([80, 20]))
    b.release(0, 64)
    assert _held(b, 0) == [4]
    for length in (1, 40, 64):
        with pytest.raises(ValueError, match="first 64 positions were released"):
            b.reserve(0, length)
    b.reserve(0, 0)
    b.reserve(0, 65)
    b.reserve(1, 40)                # the other sequence has released none
    assert _held(b, 0) == [4] and _held(b, 1) == [0, 1, 2]
    with pytest.raises(ValueError, match="released"):
        b.truncate(63)              # behind what is there
    assert b.length.tolist() == [80, 20]
    b.truncate(70)
    assert b.length.tolist() == [70, 20]
    b.truncate(0)                   # all positions forgotten: from the start again
    b.reserve(0, 40)
    assert _held(b, 0) == [0, 1, 2, 4]
    b.reserve(0, 96)
    assert _held(b, 0) == [0, 1, 2, 3, 4, 5]
    used = [i for i in b.table.flatten().tolist() if i >= 0]
    assert len(set(used)) == len(used) == 9 and len(b._free) == 3
    b.release(0, 32)
    b.release(0)
    b.reserve(0, 16)
    assert _held(b, 0) == [0]
    b.release(0, 1 << 40)           # past the table
    with pytest.raises(ValueError, match="released"):
        b.reserve(0, 96)
    b.reset()
    b.reserve(0, 96)


@pytest.mark.gpu
def test_append_behind_a_released_page(dev):
    b = DevicePagedKVBuffer(2, 1, 16, 12, 16, 6, device=dev)
    x = torch.randn(2, 20, 1, 16, device=dev)
    for i in range(2):
        b.reserve(i, 80)
    b.append(x, x, 40)
    b.release(0, 48)
    kept = [t.clone() for t in (b.k, b.v, b.length)]
    with pytest.raises(ValueError, match="first 48 positions were released"):
        b.append(x, x, 40)
    with pytest.raises(ValueError, match="released"):
        b.append(x[0], x[0], 47, None, 0)
    assert all(torch.equal(t, u) for t, u in zip(kept, (b.k, b.v, b.length)))
    b.append(x[1], x[1], 0, None, 1)
    b.append(x[0], x[0], 48, None, 0)
    assert b.length.tolist() == [68, 20]
    for i, start in ((0, 48), (1, 0)):
        k, v = b.read(start, 20, sequence=i)
        assert torch.equal(k, x[i]) and torch.equal(v, x[i])
    b.truncate(0)
    b.reserve(0, 20)
    b.append(x, x)
    assert torch.equal(b.read(0, 20)[0], x)
