"""Tree steps followed by other steps of the runner, and pages released in the middle of a prompt, on the GPU."""
import pytest
import torch

import nano_qwen_amd.utils.context as C
from nano_qwen_amd.engine import Sequence
from oracle import spans
from tests.spans import check, half_step
from tests.test_gpu_spans_use import BF, _engine, _run, _token_rows

pytestmark = pytest.mark.gpu
# two outputs of the same token: rounding of P and of the output in both, values of |v| <= 5
CLOSE = 2 * 1.02 * (2 * half_step(BF) + 5e-4) * 5


def _decode(runner, attns, seq, cuda):
    runner.sampled_token_ids_gpu[:1] = torch.tensor([seq.last_token])
    ids, pos = runner.prepare_decode([seq])
    return _run(attns, ids, pos, cuda)


@pytest.mark.parametrize("accepted", [0, 1, 3])
def test_decode_after_partial_acceptance(cuda, accepted):
    """A tree whose drafts reach two pages further than what is accepted, then decode steps, against plain decoding."""
    runner, attns = _engine(cuda, 2)
    tokens = list(range(50, 78))
    a, twin = Sequence(tokens, [7, 2, 11], 0, 28), Sequence(tokens, [20], 0, 28)
    ids, pos = runner.prepare_prefill([a, twin])
    _run(attns, ids, pos, cuda)
    for s in (a, twin):
        s.append_token(500)
    drafts = [list(range(501, 501 + 40))]    # a chain: positions 28 .. 68, three pages
    ids, pos = runner.prepare_tree([a], drafts, [list(range(40))])
    _run(attns, ids, pos, cuda)
    targets = [501 + i if i < accepted else 9 for i in range(41)]
    path, count, following = runner.commit_tree(torch.tensor(targets, device=cuda))
    runner.accept_tree([a], drafts, path, count, following)
    assert a.token_ids == tokens + [500, *range(501, 501 + accepted), 9] and a.block_table == [7, 2, 11]
    for token in (*range(501, 501 + accepted), 9):
        _decode(runner, attns, twin, cuda)
        twin.append_token(token)
    for step in range(6):    # over the edge of the first page
        if len(twin) == 33:
            twin.block_table.append(21)
        for x, y in zip(_decode(runner, attns, a, cuda), _decode(runner, attns, twin, cuda)):
            assert torch.isfinite(x).all() and (x.float() - y.float()).abs().max() <= CLOSE, step
        for s in (a, twin):
            s.append_token(700 + step)
    raw = runner.kv_cache.view(torch.uint8)
    for p in range(len(a) - 1):
        x, y = (raw[:, :, s.block_table[p // 32], p % 32] for s in (a, twin))
        assert torch.equal(x, y), p
    C.reset_context()


def test_pages_released_between_chunks(cuda):
    """A long prompt through windowed layers in chunks, pages given back after each and overwritten by their takers."""
    window, sinks, n = 40, 3, 190
    runner, attns = _engine(cuda, 2, window=window, num_sinks=sinks)
    tokens = list(range(300, 300 + n))
    s = Sequence(tokens, [9, 3, 14, 1, 22, 6])
    rows = [_token_rows(tokens, range(n), i, "cpu") for i in range(2)]
    see = spans.window_visible(torch.arange(n), n, window, sinks)
    want = [spans.attend(q, k.double(), v.double(), see, 128 ** -0.5) for q, k, v in rows]
    done, freed = 0, []
    for chunk in (32, 40, 1, 77, 39):
        s.num_cached_tokens, s.num_scheduled_tokens = done, chunk
        ids, pos = runner.prepare_prefill([s])
        outs = _run(attns, ids, pos, cuda)
        done += chunk
        for out, (ref, mag) in zip(outs, want):
            check(out, ref[done - chunk:done], mag[done - chunk:done], BF, f"to {done}")
        taken = runner.release_window_blocks(s, window, sinks)
        runner.kv_cache[:, :, taken] = float("nan")
        freed += taken
    assert done == n - 1 and freed == [3, 14, 1]    # 150 .. 189 are seen by the last token
    s.append_token(1000)
    C.reset_context()
