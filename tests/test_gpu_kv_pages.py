"""Page copies and tree commits on the GPU: bytes against the oracle's."""
import random

import pytest
import torch

from nano_qwen_amd import kernels
from oracle import spans
from tests.spans import random_tree

pytestmark = pytest.mark.gpu


def pool(shape, dtype, seed=0):
    n = 1
    for x in shape:
        n *= x
    raw = torch.randint(0, 256, (n * torch.empty((), dtype=dtype).element_size(),), dtype=torch.uint8,
                        generator=torch.Generator().manual_seed(seed))
    return raw.view(dtype).view(shape)


def same_bytes(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


@pytest.mark.parametrize("shape,dtype", [((2, 3, 9, 32, 2, 128), torch.bfloat16), ((2, 1, 7, 256, 8, 128), torch.float16),
                                         ((5, 64, 1, 16), torch.float8_e4m3fn), ((2, 2, 6, 96, 3, 20), torch.float32)])
@pytest.mark.parametrize("partial", [False, True])
def test_copy(cuda, shape, dtype, partial):
    p = pool(shape, dtype)
    nb, bs = shape[-4], shape[-3]
    dev = p.to(cuda)
    ids = random.Random(nb).sample(range(nb), nb)
    src, dst = ids[:nb // 2], ids[nb // 2:2 * (nb // 2)]
    tokens = [1 + 7 * i % bs for i in range(len(src))] if partial else None
    if partial:
        tokens[0], tokens[-1] = bs, 0
    kernels.copy_kv_blocks(dev, *(torch.tensor(x, dtype=torch.int32, device=cuda) for x in (src, dst)),
                           None if tokens is None else torch.tensor(tokens, dtype=torch.int32, device=cuda))
    raw = p.clone()
    for i, (a, b) in enumerate(zip(src, dst)):
        n = bs if tokens is None else tokens[i]
        raw.view(torch.uint8)[..., b, :n, :, :] = p.view(torch.uint8)[..., a, :n, :, :]
    assert same_bytes(dev, raw)


def test_copy_skips_bad_pairs(cuda):
    p = pool((2, 4, 32, 2, 128), torch.bfloat16)
    dev = p.to(cuda)
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)    # noqa: E731
    kernels.copy_kv_blocks(dev, t(-1, 0, 4, 2, 1), t(0, 4, 1, 2, 3), t(32, 32, 32, 32, 99))
    raw = p.clone()
    raw[:, 3] = p[:, 1]    # more tokens than a page holds: the page
    assert same_bytes(dev, raw)
    kernels.copy_kv_blocks(dev, t(), t())
    assert same_bytes(dev, raw)


@pytest.mark.parametrize("new,pre,block,shape,dtype", [
    ([8], [300], 256, (2, 2, 0, 0, 8, 128), torch.bfloat16),
    ([1, 5, 64, 0, 33, 2], [0, 31, 500, 9, 64, 1], 32, (2, 3, 0, 0, 2, 128), torch.float16),
    ([256, 100], [7, 90], 64, (2, 1, 0, 0, 1, 256), torch.bfloat16),
    ([26] * 9, list(range(9)), 32, (3, 0, 0, 1, 16), torch.float8_e4m3fn),
])
def test_commit(cuda, new, pre, block, shape, dtype):
    r = random.Random(sum(new))
    n = len(new)
    counts = [-(-(a + b) // block) for a, b in zip(new, pre)]
    nb = sum(counts) + 2
    shape = (*shape[:-4], nb, block, *shape[-2:])
    p = pool(shape, dtype)
    perm = random.Random(1).sample(range(nb), nb)
    table = torch.full((n, max(counts) + 1), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = torch.tensor(perm[at:at + c], dtype=torch.int32)
        at += c
    parents, tokens, targets, paths, nexts = [], [], [], [], []
    ref = p.clone()
    for i, (k, c) in enumerate(zip(new, pre)):
        if k == 0:
            paths.append([])
            nexts.append(-1)
            continue
        t = random_tree(r, k)
        tok = [r.randrange(4) + 2 ** 33 * r.randrange(2) for _ in t]    # few values: siblings share tokens
        tgt = [r.randrange(4) + 2 ** 33 * r.randrange(2) for _ in t]
        for v in range(k):    # mostly follow a child
            kids = [j for j, q in enumerate(t) if q == v]
            if kids and r.random() < 0.9:
                tgt[v] = tok[r.choice(kids)]
        path, nxt = spans.accepted_path(t, tok, tgt)
        spans.move_rows(ref.view(torch.uint8), table[i], c, path)
        parents += t
        tokens += tok
        targets += tgt
        paths.append(path)
        nexts.append(nxt)
    cu = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32, device=cuda)    # noqa: E731
    i64 = lambda x: torch.tensor(x, dtype=torch.int64, device=cuda)    # noqa: E731
    dev = p.to(cuda)
    args = (table.to(cuda), cu(new), cu([a + b for a, b in zip(new, pre)]), max(new))
    path, count, nxt = kernels.commit_tree(dev, *args, torch.tensor(parents, dtype=torch.int32, device=cuda),
                                           i64(tokens), i64(targets))
    assert max(len(x) for x in paths) > (1 if max(new) > 1 else 0)
    assert path.tolist() == [x + [-1] * (max(new) - len(x)) for x in paths]
    assert count.tolist() == [len(x) for x in paths] and nxt.tolist() == nexts
    assert same_bytes(dev, ref)
    # the same paths given
    again = p.to(cuda)
    back = kernels.commit_tree(again, *args, path=path, num_accepted=count)
    assert back[0] is path and back[2] is None and same_bytes(again, ref)


def test_commit_given_paths_end_where_they_do_not_rise(cuda):
    p = pool((2, 3, 32, 1, 64), torch.bfloat16)
    dev = p.to(cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)    # noqa: E731
    table, cu_q, cu_k = i32([[2, 0]]), i32([0, 6]), i32([0, 36])
    path = i32([[0, 3, 4, 4, 5, 2]])
    kernels.commit_tree(dev, table, cu_q, cu_k, 6, path=path, num_accepted=i32([6]))
    ref = spans.move_rows(p.clone(), table[0].tolist(), 30, [0, 3, 4])
    assert same_bytes(dev, ref)
    kernels.commit_tree(dev, table, cu_q, cu_k, 6, path=i32([[0, 9, 4, 4, 5, 2]]), num_accepted=i32([99]))
    assert same_bytes(dev, ref)


@pytest.mark.parametrize("most", [0, 7])
def test_commit_without_nodes(cuda, most):
    """A step in which no sequence has a node still answers for each of them."""
    p = pool((2, 2, 4, 32, 1, 64), torch.bfloat16)
    dev = p.to(cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)    # noqa: E731
    none = torch.empty(0, dtype=torch.int64, device=cuda)
    held = [torch.full((4096,), 77, dtype=torch.int32, device=cuda) for _ in range(8)]    # what new tensors then find
    del held
    path, count, nxt = kernels.commit_tree(dev, i32([[0], [1], [2]]), i32([0, 0, 0, 0]), i32([0, 9, 9, 30]), most,
                                           i32([]), none, none)
    assert path.tolist() == [[-1] * most] * 3 and count.tolist() == [0] * 3 and nxt.tolist() == [-1] * 3
    assert same_bytes(dev, p)


def test_captured_commit_and_copy(cuda):
    """One graph that accepts a tree, moves its rows and copies its page, replayed over new drafts and pools."""
    r = random.Random(4)
    shape, pre, n = (2, 2, 6, 32, 2, 64), 40, 20
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)    # noqa: E731
    dev = pool(shape, torch.float16).to(cuda)
    table, cu_q, cu_k, src, dst = i32([[3, 1]]), i32([0, n]), i32([0, pre + n]), i32([1]), i32([4])
    parents, tokens, targets = (torch.zeros(n, dtype=t, device=cuda) for t in (torch.int32, torch.int64, torch.int64))

    def step():
        got = kernels.commit_tree(dev, table, cu_q, cu_k, n, parents, tokens, targets)
        kernels.copy_kv_blocks(dev, src, dst)
        return got

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        tree = random_tree(r, n)
        tok = [r.randrange(3) for _ in tree]
        tgt = [r.randrange(3) for _ in tree]
        for v in range(n):
            kids = [j for j, q in enumerate(tree) if q == v]
            if kids:
                tgt[v] = tok[r.choice(kids)]
        p = pool(shape, torch.float16, seed=turn)
        ref = p.clone()
        for x, y in ((parents, tree), (tokens, tok), (targets, tgt)):
            x.copy_(torch.tensor(y))
        dev.copy_(p)
        graph.replay()
        path, nxt = spans.accepted_path(tree, tok, tgt)
        spans.move_rows(ref.view(torch.uint8), table[0].tolist(), pre, path)
        ref[:, :, 4] = ref[:, :, 1]
        assert out[0].tolist() == [path + [-1] * (n - len(path))] and out[1].tolist() == [len(path)]
        assert out[2].tolist() == [nxt] and same_bytes(dev, ref), turn
