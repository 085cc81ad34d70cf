"""The runner's host side around tree steps, releases and compaction (CPU)."""
import pytest
import torch

import nano_qwen_amd.utils.context as C
from nano_qwen_amd import kernels
from nano_qwen_amd.engine import ModelRunner, Sequence
from nano_qwen_amd.layers import Attention, gdn_core


def make_runner(block=32, blocks=40, layers=2):
    runner = ModelRunner(block_size=block, max_num_seqs=8, device="cpu")
    attns = torch.nn.ModuleList(Attention(4, 128, 128 ** -0.5, 2) for _ in range(layers))
    runner.allocate_kv_cache(attns, layers, blocks, 2, 128, torch.bfloat16)
    return runner


def test_decode_goes_to_the_page_of_its_position(monkeypatch):
    """A table with pages to spare (a tree step's drafts that were not accepted) decodes into the right one."""
    runner = make_runner()
    seen = {}
    monkeypatch.setattr(kernels, "prepare_decode", lambda ids, slots, lens, last, *rest: seen.update(
        lens=lens[:rest[-2]].tolist(), last=last[:rest[-2]].tolist()))
    a, b = Sequence(list(range(30)), [7, 2, 11]), Sequence(list(range(33)), [4, 5])
    runner.prepare_tree([a, b], [[1, 2, 3, 4], [1]], [[0, 0, 1, 2], [0]])
    runner.accept_tree([a, b], [[1, 2, 3, 4], [1]], torch.tensor([[0, 1, -1, -1, -1], [0, -1, -1, -1, -1]]),
                       torch.tensor([2, 1]), torch.tensor([55, 66]))
    for s, last in ((a, 7), (b, 5)):
        runner.prepare_decode([s])
        assert seen == dict(lens=[len(s)], last=[last])
    a.append_token(9)    # 33 tokens: the second page
    runner.prepare_decode([a, b])
    assert seen == dict(lens=[33, 34], last=[2, 5])
    C.reset_context()


@pytest.mark.parametrize("window,sinks", [(40, 3), (1, 0), (33, 40), (300, 1)])
def test_pages_released_between_chunks(window, sinks):
    """While a prompt is prefilled in chunks, every page that a later token sees stays in the table."""
    runner = make_runner()
    n = 150
    s = Sequence(list(range(n)), [9, 3, 14, 1, 22])
    done = 0
    for chunk in (32, 32, 20, 60, 6):
        s.num_cached_tokens, s.num_scheduled_tokens = done, chunk
        runner.prepare_prefill([s])
        assert min(C.get_context().slot_mapping.tolist()) >= 0
        done += chunk
        runner.release_window_blocks(s, window, sinks)
        for i, page in enumerate(s.block_table):    # seen by a later token, or to be written
            needed = any(j >= done or j < sinks or j > min(done, n - 1) - window for j in range(32 * i, 32 * i + 32))
            assert (page >= 0) == needed, (done, i)
    s.append_token(7)
    runner.release_window_blocks(s, window, sinks)
    assert [x >= 0 for x in s.block_table] == [32 * i < sinks or 32 * i + 31 > 150 - window for i in range(5)]
    C.reset_context()


def test_release_from_a_position():
    runner = make_runner()
    s = Sequence(list(range(200)), list(range(10, 17)))
    assert runner.release_window_blocks(s, 40, 3, position=64) == []
    assert runner.release_window_blocks(s, 40, 3, position=103) == [11]    # 64 .. 103 are seen
    assert runner.release_window_blocks(s, 40, 3) == [12, 13, 14]          # 160 .. 199
    s.num_prepared_tokens = 200
    with pytest.raises(ValueError):    # refused: nothing is prepared
        runner.prepare_tree([s, Sequence([1], [2])], [[1], [2]], [[0], [1]])
    assert s.num_prepared_tokens == 200
    t = Sequence(list(range(200)), [1])
    assert runner.release_window_blocks(t, 10) == [1]                      # no pages behind the first


def test_tree_steps_end_once(monkeypatch):
    """A step is committed once, and the pool is not compacted under it."""
    runner = make_runner()
    calls = []
    monkeypatch.setattr(kernels, "commit_tree", lambda *a, **kw: calls.append(a) or "done")
    monkeypatch.setattr(kernels, "copy_kv_blocks", lambda *a: None)
    with pytest.raises(RuntimeError, match="no tree step"):
        runner.commit_tree(torch.zeros(3, dtype=torch.int64))
    a, b = Sequence(list(range(30)), [7, 2]), Sequence([1, 2], [9])
    runner.prepare_tree([a], [[5, 6]], [[0, 1]])
    with pytest.raises(RuntimeError, match="open"):
        runner.compact([a, b])
    assert a.block_table == [7, 2]
    assert runner.commit_tree(torch.zeros(3, dtype=torch.int64)) == "done" and len(calls) == 1
    with pytest.raises(RuntimeError, match="no tree step"):
        runner.commit_tree(torch.zeros(3, dtype=torch.int64))
    # the next sequences' step is prepared before this one's are brought up to date
    runner.prepare_tree([b], [[5]], [[0]])
    result = torch.tensor([[0, 1]]), torch.tensor([2]), torch.tensor([8])
    runner.accept_tree([a], [[5, 6]], *result)
    runner.commit_tree(torch.zeros(2, dtype=torch.int64))
    assert len(calls) == 2
    # a caller that commits through kernels.commit_tree
    runner.prepare_tree([b], [[5]], [[0]])
    runner.accept_tree([b], [[5]], *result)
    assert runner.compact([a, b]) == 3 and runner.tree is None
    # a call that is refused leaves the step open
    runner.prepare_tree([a], [[5, 6]], [[0, 1]])
    monkeypatch.undo()
    with pytest.raises(RuntimeError, match="device"):
        runner.commit_tree(torch.zeros(3, dtype=torch.int64))
    assert runner.tree is not None
    C.reset_context()


def test_recurrent_layers_refuse_trees():
    """A tree step looks like a prefill, but its nodes are no sequence."""
    runner = make_runner()
    x = torch.zeros(3, 8)
    runner.prepare_tree([Sequence([1], [0])], [[5, 6]], [[0, 0]])
    with pytest.raises(RuntimeError, match="trees"):
        gdn_core(None, x, x, x, x, torch.zeros(1, dtype=torch.int32), cu_seqlens=C.get_context().cu_seqlens_q)
    C.reset_context()
    with pytest.raises(AttributeError):    # past the check
        gdn_core(None, x, x, x, x, torch.zeros(1, dtype=torch.int32))
