"""Tree speculation at its edges: rows that are not finite, operators in a row, sums that nearly tie, lengths at the ends of
their types."""
import numpy as np
import pytest
import torch

from hipml_b200 import _lib, api
from tests import tree_reference as R
from tests.test_gpu_tree import Step, _dev, _ints, _spoil, status  # noqa: F401 (status: every test leaves the device's clear)

pytestmark = pytest.mark.gpu


# ---- attention ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", [(0,), (1,), (0, 1)], ids=["k", "v", "kv"])
def test_a_run_of_rows_that_are_not_finite(dim, kv_dtype, value, which):
    """Of two roots behind 128 rows one's own row is all that it sees of the last run; where that is not finite, neither is
    the node. The other root does not see it."""
    step = Step(1, kv_dtype, [(128, 2, [-1, -1])], 2, heads=4, kv=2, dim=dim)
    for w in which:
        _spoil(step, w, 0, 128, value)
    step.upload()
    step.call()
    got = step.out.cpu().numpy().reshape(2, 4, dim)
    want, bound = R.attention(step.caches, 0, 128, 2, [-1, -1], step.q[0].reshape(2, 4, dim), 4, step.scale)
    assert not np.isfinite(got[0]).any()
    assert (np.abs(got[1] - want[1]) <= bound[1]).all()


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
@pytest.mark.parametrize("which", [0, 1], ids=["k", "v"])
def test_a_whole_tile_of_rows_that_are_not_finite(dim, kv_dtype, which):
    """64 rows of the prefix of one of two slots; of many runs exactly one has nothing else."""
    step = Step(2, kv_dtype, [(512, 3, R.chain(3)), (300, 2, R.chain(2))], 3, heads=4, kv=2, dim=dim)
    for row in range(128, 192):
        _spoil(step, which, 0, row, float("nan"))
    step.upload()
    step.call()
    got = step.out.cpu().numpy().reshape(2, 3, 4, dim)
    assert not np.isfinite(got[0]).any()
    want, bound = R.attention(step.caches, 1, 300, 2, R.chain(2), step.q[1].reshape(3, 4, dim), 4, step.scale)
    assert (np.abs(got[1, :2] - want) <= bound).all()


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
@pytest.mark.parametrize("base", [40, 128])
def test_keys_whose_scores_would_be_minus_infinity(dim, kv_dtype, base):
    """Queries of one sign and a key of -infinity: the row does not leave with a weight of 0, the node is not finite."""
    step = Step(3, kv_dtype, [(base, 2, [-1, -1])], 2, heads=4, kv=2, dim=dim)
    step.q[:] = np.abs(step.q) + 0.5
    step.caches.put(0, 0, base, np.ones((2, 1, dim)))
    _spoil(step, 0, 0, base, -float("inf"))
    if kv_dtype == 2:   # (its codes count from -8: all of them above 0)
        codes = step.caches.rows(0, 0)[:, base].reshape(2, -1, R.ROW_BYTES[2])[:, :, 2:]
        codes[:] = 0xFF
    step.upload()
    step.call()
    got = step.out.cpu().numpy().reshape(2, 4, dim)
    want, bound = R.attention(step.caches, 0, base, 2, [-1, -1], step.q[0].reshape(2, 4, dim), 4, step.scale)
    assert not np.isfinite(got[0]).any()
    assert (np.abs(got[1] - want[1]) <= bound[1]).all()


def test_ends_at_the_edge_of_their_type():
    """The end words of pos are any 32-bit numbers: a negative end is an empty slot, an end past the cache the cache's."""
    low, high = -(1 << 31), (1 << 31) - 1
    tree = R.chain(4)
    for dim in (64, 256):
        step = Step(4, 1, [(70, 0, tree), (1, 0, tree), (60, 4, tree), (0, 4, tree), (70, 0, tree)], 4, heads=4, kv=2, dim=dim,
                    stride=70)
        step.parents[:] = tree
        step.dparents = _dev(step.parents)
        step.pos = _ints([[70, low], [1, low], [60, 64], [low, 4], [high, low]])
        step.run()
        step.pos = _ints([[70, high], [1, low + 5], [60, 64], [low, 4], [high, high]])
        step.run()
    path, count, following = (torch.full((n,), 9, dtype=torch.int32, device="cuda") for n in (12, 3, 3))
    api.tree_verify(_ints([[5, low], [high, low], [1, low + 3]]), _ints([tree] * 3), _ints([[0, 1, 2, 3]] * 3),
                    torch.ones(3, 4, 5, device="cuda"), None, torch.zeros(3, 4, device="cuda"), path, count, following, 4, 3, 5)
    assert (torch.cat([path, count, following]) == 9).all()


def test_a_cache_of_as_many_rows_as_an_int_counts():
    """2^31 - 1 rows of 18 bytes; the last run ends within a tile of the largest int. Keys are 0, so every row counts alike."""
    stride, live, dim = (1 << 31) - 1, 3, 32
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 39 GB")
    cache = torch.zeros(stride, 18, dtype=torch.uint8, device="cuda")
    base = stride - live
    row = torch.from_numpy(np.frombuffer(np.float16(1.0).tobytes() + bytes([0x9F] * 16), dtype=np.uint8).copy()).cuda()
    cache[base] = row     # low nibbles 15 (values 7), high ones 9 (values 1)
    q = torch.zeros(1, live, dim, device="cuda")
    out = torch.empty(1, live, dim, device="cuda")
    ws = torch.empty(api.attn_tree_workspace_bytes(1, 1, dim, live, 1), dtype=torch.uint8, device="cuda")
    api.attn_tree(_ints([[base, stride]]), _ints([[-1, -1, 0]]), q, cache, cache, out, 1, 1, dim, stride, 1.0, live, 1, 0, ws,
                  kv_dtype=2)
    got = out.cpu().numpy().reshape(live, dim).astype(np.float64)
    value = np.r_[np.full(16, 7.0), np.full(16, 1.0)]
    # (scores are 0: a weight of 1 a row; whole numbers below 2^24 in each of the runs, and then at most 42 sums one after
    # another, a reciprocal and a product, each rounded by 2^-24 of itself: less than 2^-18)
    for node, rows, seen in ((0, base + 1, 1), (1, base + 1, 0), (2, base + 2, 1)):
        assert (np.abs(got[node] - seen * value / rows) <= 2.0 ** -18 * value / rows).all()


# ---- the operators in a row --------------------------------------------------------------------------------------

def test_a_slot_that_goes_idle_between_steps():
    """Verification leaves an idle slot's path and count as the step before left them; the kept path is not theirs to move."""
    rng = np.random.default_rng(5)
    nodes, vocab, kv, dim, stride = 5, 20, 2, 64, 40
    target = torch.zeros(2, nodes, vocab, device="cuda")
    tokens = np.array([[0, 3, 4, 5, 6]] * 2)
    parents = [[-1, 0, 0, 2, 3]] * 2
    target[:, 0, 4] = target[:, 2, 5] = target[:, 3, 1] = 1.0    # path 0, 2, 3
    path, count, following = (torch.full(s, -7, dtype=torch.int32, device="cuda") for s in ((2, nodes), (2,), (2,)))
    host = [rng.integers(0, 256, (2, kv, stride, dim // 32 * 34), dtype=np.uint8) for _ in range(2)]
    caches = [_dev(h) for h in host]

    def step(lives, base):
        pos = _ints([[b, b + n] for b, n in zip(base, lives)])
        api.tree_verify(pos, _ints(parents), _ints(tokens.tolist()), target, None, torch.zeros(2, nodes, device="cuda"), path,
                        count, following, nodes, 2, vocab)
        api.kv_path_keep(pos, path, count, caches[:1], caches[1:], kv, dim, stride, nodes, 2, kv * stride * (dim // 32 * 34))

    def keep(slot, base):
        for h in host:
            h[slot, :, base:base + 3] = h[slot, :, [base, base + 2, base + 3]].swapaxes(0, 1)

    step((5, 5), (10, 4))
    keep(0, 10), keep(1, 4)
    step((0, 5), (13, 7))       # slot 0 idles
    keep(1, 7)
    step((0, 0), (13, 10))
    step((4, 0), (13, 10))
    keep(0, 13)
    assert api.check_device_status() == 0
    assert count.tolist() == [3, 3] and path[:, :3].tolist() == [[0, 2, 3]] * 2
    for h, c in zip(host, caches):
        assert np.array_equal(h, c.cpu().numpy())


@pytest.mark.parametrize("looked_up", [False, True], ids=["drawn", "looked up"])
def test_trees_that_cross_the_end_of_the_cache(looked_up):
    """Attention, verification and the kept path agree on which nodes the cache has: the last two are not among them, although
    their tokens would be kept (their target rows hold what nobody computed)."""
    nodes, vocab, kv, dim, stride, base = 6, 30, 2, 64, 50, 46
    parents = R.chain(nodes)
    step = Step(7, 1, [(base, 4, parents)], nodes, heads=4, kv=kv, dim=dim, stride=stride)
    step.parents[:] = parents
    step.dparents, step.pos = _dev(step.parents), _ints([[base, base + nodes]])
    step.run()
    tokens = [0, 1, 2, 3, 4, 5]
    target = np.full((1, nodes, vocab), np.nan, dtype=np.float32)
    target[0, :4] = 0.5 / vocab
    for i in range(4):
        target[0, i, i + 1] = 0.5
    draft = None if looked_up else np.full((1, nodes, vocab), 1.0 / vocab, dtype=np.float32)
    u = np.full((1, nodes), 0.25, dtype=np.float32)
    path, count, following = (torch.full(s, -7, dtype=torch.int32, device="cuda") for s in ((1, nodes), (1,), (1,)))
    api.tree_verify(step.pos, step.dparents, _ints([tokens]), _dev(target), None if looked_up else _dev(draft), _dev(u), path,
                    count, following, nodes, 1, vocab, stride=stride)
    want, token = R.verify(parents, tokens, target[0], None if looked_up else draft[0], u[0], 4)
    assert want == [0, 1, 2, 3]
    assert path[0].tolist() == want + [-1, -1] and count.tolist() == [4] and following.tolist() == [token]
    api.kv_path_keep(step.pos, path, count, [step.dk], [step.dv], kv, dim, stride, nodes, 1, 0)
    assert api.check_device_status() == 0


# ---- sums --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rejected", [False, True], ids=["root", "rejected"])
@pytest.mark.parametrize("drawn", [False, True], ids=["looked up", "drawn"])
@pytest.mark.parametrize("short", [False, True], ids=["past", "short"])
def test_the_longest_rows_where_the_bar_lies_next_to_a_running_sum(rejected, drawn, short):
    """2^20 tokens, whole numbers of 2^-61 whose running sum over the first half is 2^-43 of the whole past half of the whole,
    or short of it. The first 32 values of every 4,096 are large and the rest lie 2^-25 below them, in the second half by a
    little less, which a long running error in 32 bits loses each time.

    Sums are exact to less than 2^-43 of what is summed: the bar (half of the whole) and the running sum (as much) together
    are less than 2^-43 of the whole off."""
    vocab, half, gone = 1 << 20, 1 << 19, (1 << 19) + 100
    units = np.full(vocab, 1 << 23, dtype=np.int64)
    units[half:] += 31
    units.reshape(-1, 4096)[:, :32] = 1 << 48
    units[gone] = 0   # the rejected child's token
    off = int(units.sum()) >> 43
    over = int(units[half:].sum()) - int(units[:half].sum()) - (2 * off if short else -2 * off)
    for at in range(vocab - 1, half, -1):   # the last tokens give what the second half has too much
        less = min(over, int(units[at]))
        units[at] -= less
        over -= less
        if over == 0:
            break
    row = (units * 2.0 ** -61).astype(np.float32)
    assert over == 0 and np.array_equal(row.astype(np.float64) * 2.0 ** 61, units)
    whole, front = int(units.sum()), int(units[:half].sum())
    assert (2 * front > whole) == (not short) and whole >> 44 <= abs(2 * front - whole) // 2 <= whole >> 42
    want = half if short else half - 1
    target = _dev(np.stack([row, row])[None])
    draft = None
    if drawn:
        draft = torch.zeros(1, 2, vocab, device="cuda")
        draft[0, 0, gone] = 1.0
    path, count, following = (torch.full(s, -7, dtype=torch.int32, device="cuda") for s in ((1, 2), (1,), (1,)))
    api.tree_verify(_ints([[3, 5 if rejected else 4]]), _ints([[-1, 0]]), _ints([[0, gone]]), target, draft,
                    torch.full((1, 2), 0.5, device="cuda"), path, count, following, 2, 1, vocab)
    assert count.tolist() == [1] and path.tolist() == [[0, -1]]
    assert following.tolist() == [want]


# ---- rotated rows ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
def test_a_captured_step_of_a_branching_tree_with_rotated_rows(kv_dtype):
    """Node i's row is rotated for position base + depth(i) and lies at base + i: the front end is called once per node, whose
    position and row are read on the device. What the step leaves is what the kept tokens as a chain make, byte for byte, for
    every base and tree that the captured step is replayed with."""
    heads, kv, dim, n_rot, nodes, stride, vocab = 24, 4, 256, 64, 9, 400, 50
    theta, eps = 1e6, 1e-6
    rng = np.random.default_rng(90)

    def floats(*shape):
        return _dev(rng.standard_normal(shape).astype(np.float32))

    qg, k, v = floats(nodes, heads * 2 * dim), floats(nodes, kv * dim), floats(nodes, kv * dim)
    qw, kw = floats(dim), floats(dim)
    q, out = (torch.zeros(1, nodes, heads * dim, device="cuda") for _ in range(2))
    fresh = R.Caches(kv_dtype, 1, kv, dim, stride, fill=0)
    caches = [_dev(b) for b in fresh.bytes]
    ids, steps = torch.zeros(nodes, 4, dtype=torch.int32, device="cuda"), torch.zeros(nodes, 8, dtype=torch.int32, device="cuda")
    pos, parents = _ints([[0, 0]]), _ints([[-1] * nodes])
    tokens, uniform = _ints([list(range(nodes))]), torch.zeros(1, nodes, device="cuda")
    target = torch.zeros(1, nodes, vocab, device="cuda")
    path, count, following = torch.zeros(1, nodes, dtype=torch.int32, device="cuda"), _ints([0]), _ints([0])
    ws = torch.empty(api.attn_tree_workspace_bytes(heads, kv, dim, nodes, 1), dtype=torch.uint8, device="cuda")

    def append(pair, token, to_q, at, step):
        """One token's query and row, at position ids `at` and cache row step[0]."""
        gate = torch.empty(heads * dim, device="cuda")
        if kv_dtype == 1:
            api.attn_front_append_q8(qg[token], k[token], v[token], to_q, gate, qw, kw, *pair, heads, kv, dim, n_rot, theta, eps,
                                     stride=stride, pos=at, step=step)
            return
        row = k[token].clone()   # (rotated in place)
        api.attn_front(qg[token], to_q, gate, row, qw, kw, heads, kv, dim, n_rot, None, at, theta, eps)
        if kv_dtype == 2:
            api.kv_encode(step, row, v[token], *pair, kv, dim, stride, dtype=1)
        else:
            api.kv_append_f32(step, pair[0].view(torch.float32), pair[1].view(torch.float32), row, v[token], kv * dim)

    def step():
        for i in range(nodes):
            append(caches, i, q[0, i], ids[i], steps[i])
        api.attn_tree(pos, parents, q, *caches, out, heads, kv, dim, stride, dim ** -0.5, nodes, 1, 0, ws, kv_dtype=kv_dtype)
        api.tree_verify(pos, parents, tokens, target, None, uniform, path, count, following, nodes, 1, vocab, stride=stride)
        api.kv_path_keep(pos, path, count, caches[:1], caches[1:], kv, dim, stride, nodes, 1, 0, kv_dtype=kv_dtype)

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for base, tree, kept in ((100, [-1, 0, 0, 1, 2, 2, 5, 5, 3], [0, 2, 5, 7]), (391, [-1, 0, 1, 1, 1, 4, 4, 6, 0], [0, 1, 4, 6, 7]),
                             (0, R.star(nodes), [0, 8])):
        depth = [len(R.sees(tree, i)) - 1 for i in range(nodes)]
        ids.copy_(_ints([[base + d] * 4 for d in depth]))
        steps.copy_(_ints([[base + i] + [0] * 7 for i in range(nodes)]))
        pos.copy_(_ints([[base, base + nodes]]))
        parents.copy_(_ints([tree]))
        target.fill_(0.0)
        for a, b in zip(kept, kept[1:] + [40]):
            target[0, a, b] = 1.0   # (node b's token is b)
        # a prefix; the kept tokens behind it as a chain, and the step over it
        prefix = R.Caches(kv_dtype, 1, kv, dim, stride, fill=0)
        if base:
            prefix.fill(rng, 0, base)
        chain = [_dev(b) for b in prefix.bytes]
        for c, b in zip(caches, chain):
            c.copy_(b)
        n = len(kept)
        chain_q = torch.zeros(1, n, heads * dim, device="cuda")
        for i, token in enumerate(kept):
            append(chain, token, chain_q[0, i], _ints([base + i] * 4), _ints([base + i] + [0] * 7))
        graph.replay()
        torch.cuda.synchronize()
        assert path[0, :n].tolist() == kept and count.tolist() == [n] and following.tolist() == [40]
        shape = (stride, kv, dim * 4) if kv_dtype == 0 else (kv, stride, fresh.row)
        for c, want in zip(caches, chain):
            c, want = (x.view(torch.uint8).view(shape) for x in (c, want))
            assert torch.equal(c[:base + n], want[:base + n]) if kv_dtype == 0 else torch.equal(c[:, :base + n], want[:, :base + n])
        at = torch.tensor(kept, device="cuda")
        assert torch.equal(q[0, at], chain_q[0])
        # the chain's attention by the same kernel, whose runs are others (both within their bounds of the definition)
        chain_out = torch.zeros(1, n, heads * dim, device="cuda")
        api.attn_tree(_ints([[base, base + n]]), _ints([R.chain(n)]), chain_q, *chain, chain_out, heads, kv, dim, stride, dim ** -0.5,
                      n, 1, 0, torch.empty_like(ws), kv_dtype=kv_dtype)
        assert float((chain_out[0] - out[0, at]).abs().max()) <= 4e-5


def test_the_status_names_what_was_wrong():
    step = Step(10, 1, [(20, 3, [-1, 0, 5])], 3, heads=2, kv=1, dim=64)
    step.call()
    with pytest.raises(_lib.HipmlError, match="no earlier node.*41"):
        api.check_device_status()
    cache = torch.zeros(2, 30, 68, dtype=torch.uint8, device="cuda")
    api.kv_path_keep(_ints([[20, 23]]), _ints([[1, 0, -1]]), _ints([2]), [cache], [cache.clone()], 2, 64, 30, 3, 1, 0)
    with pytest.raises(_lib.HipmlError, match="does not ascend.*42"):
        api.check_device_status()
