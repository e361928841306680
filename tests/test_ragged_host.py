"""Host side of the ragged path (CPU): padded batches taken apart, all-or-nothing growth of the block tables, the
scheduler's packed prefill, and the arguments that ``verify`` and ``prefill_ragged`` turn down."""

import pytest
import torch

from microgen_b200.backends.b200 import B200QuantizedBackend, PagedKVCache
from microgen_b200.model_spec import ModelSpec
from microgen_b200.runtime.paged_kv import PagedKVCacheAllocator
from microgen_b200.scheduler import BatchedScheduler
from tests.test_scheduler import FakeBackend, V, _req, stream


class _Eng:
    max_batch, max_blocks = 4, 4


def _backend(num_blocks=8):
    """A backend without a device: its allocator and limits only."""
    be = object.__new__(B200QuantizedBackend)
    be.engine, be.allocator = _Eng(), PagedKVCacheAllocator(num_blocks=num_blocks)
    be.max_batch, be.max_seq_len = 4, 64
    be.spec = ModelSpec(family="llama", hidden=128, layers=1, heads=4, kv_heads=2, head_dim=32, inter=256, vocab=50,
                        eps=1e-5)
    return be


def test_unpadded_rows():
    ids = torch.tensor([[0, 0, 5, 6], [7, 8, 0, 0], [0, 9, 0, 0], [1, 2, 3, 4]])
    mask = torch.tensor([[0, 0, 1, 1], [1, 1, 0, 0], [0, 1, 0, 0], [1, 1, 1, 1]])
    assert B200QuantizedBackend._unpadded(ids, mask) == [[5, 6], [7, 8], [9], [1, 2, 3, 4]]
    assert B200QuantizedBackend._unpadded([3, 4], [0, 1]) == [[4]]


@pytest.mark.parametrize("ids,mask", [([[1, 2, 3]], [[1, 0, 1]]), ([[1, 2]], [[0, 0]]), ([[1, 2], [3, 4]], [[1, 0, 1], [1, 1, 1]])])
def test_unpadded_refusals(ids, mask):
    with pytest.raises(ValueError):
        B200QuantizedBackend._unpadded(torch.tensor(ids), torch.tensor(mask))


def test_tables_grow_all_or_none():
    be = _backend(num_blocks=6)
    tabs = [be.allocator.allocate_sequence("a", 15), be.allocator.allocate_sequence("b", 16)]
    assert be._grow(tabs, [2, 17]) == [15, 16]
    assert [t.num_tokens for t in tabs] == [17, 33] and [t.num_blocks() for t in tabs] == [2, 3]
    free = be.allocator.get_num_free_blocks()
    with pytest.raises(MemoryError):
        be._grow(tabs, [16, 16])  # two more blocks, and one is free
    assert [t.num_tokens for t in tabs] == [17, 33] and be.allocator.get_num_free_blocks() == free
    with pytest.raises(ValueError):
        be._grow(tabs, [0, 32])   # past max_seq_len
    be._shrink(tabs, [15, 17])
    assert [t.num_tokens for t in tabs] == [15, 17] and [t.num_blocks() for t in tabs] == [1, 2]


def test_prefill_ragged_and_verify_refuse_on_the_host():
    be = _backend()
    for bad in ([], [[1], []], [[1]] * 5):
        with pytest.raises(ValueError):
            be.prefill_ragged(bad)
    cache = PagedKVCache(be.allocator)
    with pytest.raises(ValueError):
        be.verify(torch.tensor([1]), [[2]], cache)  # nothing prefilled
    cache.tables = [be.allocator.allocate_sequence("a", 3)]
    for toks, drafts in (([1, 2], [[3]]), ([1], [[3], [4]]), ([1], [[50]]), ([1], [[-1]])):
        with pytest.raises(ValueError):
            be.verify(torch.tensor(toks), drafts, cache)
    assert cache.tables[0].num_tokens == 3


class _PackedBackend(FakeBackend):
    def prefill_ragged(self, prompts):
        cache = PagedKVCache(self.allocator)
        cache.tables = [self.allocator.allocate_sequence(f"seq{i}", len(p)) for i, p in enumerate(prompts)]
        self.calls.append(("prefill_ragged", len(prompts), 0))
        return self._logits([p[-1] for p in prompts], [len(p) - 1 for p in prompts]), cache


def test_scheduler_packs_prompts_of_different_lengths():
    be = _PackedBackend(num_blocks=256)
    sch = BatchedScheduler(be, max_batch_size=4, packed_prefill=True)
    reqs = [_req(i, [(i * 13 + j) % V for j in range(5 + 7 * i)], 6 + 3 * i) for i in range(7)]
    for r in reqs:
        sch.add_request(r)
    sch.run_until_complete()
    for r in reqs:
        assert r.generated_token_ids == stream(r.prompt_ids, r.max_new_tokens)
    assert be.calls[0] == ("prefill_ragged", 4, 0)  # four lengths, one call
    assert not any(c[0] == "prefill" for c in be.calls)
    assert be.allocator.get_num_allocated_blocks() == 0
