"""What PagedBatch and the calls that take it check on the host, with stand-ins for device tensors: nothing here needs a GPU."""
import copy

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


def test_a_copy_of_a_batch_has_addresses_of_its_own():
    b = batch()
    b.dtype = fa.F32
    other = copy.copy(b)
    assert all(getattr(other, n) is getattr(b, n) for n in fa.PagedBatch.TENSORS) and other.dtype == fa.F32
    old = b.raw.page_counts
    other.page_counts = Ints(2, at=0x7770)
    assert b.raw.page_counts == old and other.raw.page_counts == 0x7770 and b.page_counts.data_ptr() == old


# ---- tensors of another device: the kernels would take their addresses ------------------------------

class Values(Ints):
    def __init__(self, *shape, dtype=torch.bfloat16, device=0):
        super().__init__(*shape, dtype=dtype, device=device)

    @property
    def nbytes(self):
        return self.numel() * torch.empty(0, dtype=self.dtype).element_size()


def context(device=0):
    """A context that has only got as far as its device: what is refused is refused before the library is called."""
    c = fa.Context.__new__(fa.Context)
    c.device, c.h = device, None
    return c


def calls(c, b, odd, d=0):
    """(tensors, call) of each entry point; the tensor number `odd` is on another device."""
    def on(tensors):
        made = [t(device=d + (i == odd)) for i, t in enumerate(tensors)]
        return made
    i = lambda *n: (lambda device: Ints(*n, device=device))  # noqa: E731
    v = lambda *n: (lambda device: Values(*n, device=device))  # noqa: E731
    out = lambda device: Values(4096, dtype=torch.uint8, device=device)  # noqa: E731
    cfg = fa.config(True)
    return {
        "reserve": ([i(2), i(3), i(6), i(6), i(6), i(2), i(1), i(2)],
                    lambda x: c.paged_batch_reserve(b, x[0], 6, x[1], x[2], x[3], x[4], x[5], x[6], x[7])),
        "release": ([i(2), i(2), i(1)], lambda x: c.paged_batch_release(b, *x)),
        "write": ([i(3), i(3), v(3, 128), v(3, 128), v(32, 128), v(32, 128)], lambda x: c.paged_kv_write(2, 64, x[0], x[1], 1e4, *x[2:])),
        "tree": ([i(3), i(3), i(3, 1), v(3, 256), v(32, 128), v(32, 128), out],
                 lambda x: c.decode_paged_tree(b, 4, 2, 64, 3, 9, x[0], x[1], x[2], cfg, 1e4, *x[3:])),
        "accept": ([i(2, 3), i(2), i(2), v(32, 128), v(32, 128)], lambda x: c.paged_kv_accept(b, 2, 64, *x)),
    }, on


@pytest.mark.parametrize("name", ["reserve", "release", "write", "tree", "accept"])
@pytest.mark.parametrize("device", [0, 1])
def test_tensors_of_another_device_than_the_context_s_are_refused(name, device):
    c, b = context(device), batch(device=device)
    for odd in range(len(calls(c, b, None)[0][name][0])):
        table, on = calls(c, b, odd, device)
        tensors, call = table[name]
        with pytest.raises(fa.FlatAttentionError) as e:
            call(on(tensors))
        assert e.value.kind == "UnsupportedShape" and f"is on cuda:{device + 1}" in e.value.detail, odd


@pytest.mark.parametrize("name", ["reserve", "release", "tree", "accept"])
def test_a_batch_of_another_device_than_the_context_s_is_refused(name):
    c, b = context(0), batch(device=1)
    table, on = calls(c, b, None)
    with pytest.raises(fa.FlatAttentionError) as e:
        table[name][1](on(table[name][0]))
    assert e.value.kind == "UnsupportedShape" and "the batch is on cuda:1" in e.value.detail


def test_the_tensors_of_a_batch_are_on_one_device():
    assert batch(device=3).device == 3
    with pytest.raises(fa.FlatAttentionError) as e:
        batch(free_count=Ints(1, device=1))
    assert e.value.kind == "UnsupportedShape" and "free_count is on cuda:1" in e.value.detail
    b = batch()
    with pytest.raises(fa.FlatAttentionError):
        b.context_lens = Ints(2, device=1)
    with pytest.raises(AttributeError):
        b.device = 1


# ---- shapes that the number of elements alone does not tell ------------------------------------------

def test_a_page_table_with_rows_of_another_length_is_refused():
    """Row s would be read from the middle of another one."""
    assert batch(page_tables=Ints(6)).raw.page_tables == 0x1000  # flat: as many as there have to be
    assert batch(page_tables=Ints(5, 3)).raw.page_tables == 0x1000  # rows that the batch does not use
    for shape in ((2, 4), (3, 2), (2, 1, 6)):
        with pytest.raises(fa.FlatAttentionError) as e:
            batch(page_tables=Ints(*shape))
        assert e.value.kind == "LengthMismatch"


def test_a_mask_without_words_is_refused():
    """An empty tensor has the address 0, which is the call without a mask."""
    c, b = context(), batch()
    with pytest.raises(fa.FlatAttentionError) as e:
        c.decode_paged_tree(b, 4, 2, 64, 3, 9, Ints(3), Ints(3), Ints(3, 0, at=0), fa.config(True), 1e4, Values(3, 256), Values(32, 128), Values(32, 128),
                            Values(4096, dtype=torch.uint8))
    assert e.value.kind == "LengthMismatch"
