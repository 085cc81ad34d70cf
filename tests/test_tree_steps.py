"""The runner's host side around tree steps, releases and compaction (CPU)."""
import torch

import nano_qwen_amd.utils.context as C
from nano_qwen_amd import kernels
from nano_qwen_amd.engine import ModelRunner, Sequence
from nano_qwen_amd.layers import Attention


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
