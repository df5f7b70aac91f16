"""What PagedBatch and the calls that take it check on the host, with stand-ins for device tensors: nothing here needs a GPU."""
import pytest
import torch

from __graft_entry__ import load_package

fa = load_package()


class Ints:
    """Looks like a contiguous int32 CUDA tensor."""

    def __init__(self, *shape, at=0x1000, dtype=torch.int32, device=0, contiguous=True):
        self.shape, self.at, self.dtype, self.device_index, self.contiguous = tuple(shape), at, dtype, device, contiguous
        self.is_cuda = device >= 0

    def numel(self):
        return int(torch.Size(self.shape).numel())

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return self.contiguous

    def get_device(self):
        return self.device_index

    def data_ptr(self):
        return self.at


def batch(S=2, page=4, pages=8, most=3, device=0, **given):
    parts = dict(page_tables=Ints(S, most, at=0x1000, device=device), page_counts=Ints(S, at=0x2000, device=device),
                 context_lens=Ints(S, at=0x3000, device=device), free_pages=Ints(pages, at=0x4000, device=device),
                 free_count=Ints(1, at=0x5000, device=device))
    return fa.PagedBatch(S, page, pages, most, **{**parts, **given})


@pytest.mark.parametrize("name", ["page_tables", "page_counts", "context_lens", "free_pages", "free_count"])
def test_a_tensor_that_is_replaced_is_the_one_the_calls_use(name):
    b = batch()
    assert getattr(b.raw, name) == getattr(b, name).data_ptr()
    new = Ints(*getattr(b, name).shape, at=0xabc0)
    setattr(b, name, new)
    assert getattr(b, name) is new and getattr(b.raw, name) == 0xabc0
    assert {getattr(b.raw, other) for other in fa.PagedBatch.TENSORS} >= {0xabc0} and sum(getattr(b.raw, o) == 0xabc0 for o in fa.PagedBatch.TENSORS) == 1


@pytest.mark.parametrize("name", ["page_tables", "page_counts", "context_lens", "free_pages", "free_count"])
def test_a_tensor_that_does_not_fit_is_refused_and_the_old_one_stays(name):
    b = batch()
    old = getattr(b, name)
    n = old.numel()
    for kind, bad in (("BufferTooSmall", Ints(n - 1)), ("UnsupportedDtype", Ints(n, dtype=torch.int64)), ("UnsupportedShape", Ints(n, contiguous=False)),
                      ("UnsupportedShape", Ints(n, device=-1)), ("NullPointer", None)):
        with pytest.raises(fa.FlatAttentionError) as e:
            setattr(b, name, bad)
        assert e.value.kind == kind
        assert getattr(b, name) is old and getattr(b.raw, name) == old.data_ptr()


@pytest.mark.parametrize("name", ["num_seqs", "page_size", "physical_pages", "max_pages_per_seq"])
def test_the_sizes_of_a_batch_are_fixed(name):
    b = batch()
    with pytest.raises(AttributeError):
        setattr(b, name, 1)
    assert getattr(b, name) == getattr(b.raw, name)
