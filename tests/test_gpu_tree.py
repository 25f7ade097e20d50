"""Tree speculation on the device against its rules in 64 bits (tests/tree_reference.py)."""
import numpy as np
import pytest
import torch

from hipml_b200 import _lib, api
from tests import tree_reference as R

pytestmark = pytest.mark.gpu

CANARY = 12345.0


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True)
def status():
    """Every test leaves the device status clear."""
    yield
    assert api.check_device_status() == 0


def _status(code):
    """A kernel has reported `code` (reading clears it)."""
    with pytest.raises(_lib.HipmlError, match=str(code)):
        api.check_device_status()


def _at_offset(a, offset):
    """The bytes of `a` on the device, `offset` bytes past a 256-byte boundary."""
    raw = np.ascontiguousarray(a).view(np.uint8).ravel()
    room = torch.zeros(raw.size + offset, dtype=torch.uint8, device="cuda")
    room[offset:] = _dev(raw)
    return room[offset:]


# ---- attention ---------------------------------------------------------------------------------------------------

class Step:
    """A drafted step of several slots on the device."""

    def __init__(self, seed, kv_dtype, shapes, nodes, heads=24, kv=4, dim=256, stride=None, pad=0, q_scale=1.5, k_scale=1.0,
                 v_scale=1.0, offset=0):
        rng = np.random.default_rng(seed)
        self.shapes, self.nodes, self.heads = shapes, nodes, heads
        self.scale = dim ** -0.5
        stride = max(b + n for b, n, _ in shapes) + 3 if stride is None else stride
        self.caches = c = R.Caches(kv_dtype, len(shapes), kv, dim, stride, pad=pad)
        for s, (base, live, _) in enumerate(shapes):
            c.fill(rng, s, base + live, k_scale, v_scale)
        self.q = (q_scale * rng.standard_normal((len(shapes), nodes, heads * dim))).astype(np.float32)
        self.parents = np.full((len(shapes), nodes), 1 << 20, dtype=np.int32)   # (of dead nodes: not looked at)
        for s, (_, live, parents) in enumerate(shapes):
            self.parents[s, :live] = parents[:live]
        self.offset = offset
        self.upload()

    def upload(self):
        c = self.caches
        self.dk, self.dv = (_at_offset(b, self.offset) for b in c.bytes)
        self.dq, self.dparents = _dev(self.q), _dev(self.parents)
        self.pos = _ints([[b, b + n] for b, n, _ in self.shapes])
        self.out = torch.full((len(self.shapes), self.nodes, self.heads * c.dim), CANARY, device="cuda")
        self.workspace = torch.full((api.attn_tree_workspace_bytes(self.heads, c.kv, c.dim, self.nodes, len(self.shapes)) // 4,),
                                    float("nan"), device="cuda")

    def call(self, **other):
        c = self.caches
        a = dict(pos=self.pos, parents=self.dparents, q=self.dq, k=self.dk, v=self.dv, out=self.out, workspace=self.workspace)
        a.update(other)
        api.attn_tree(a["pos"], a["parents"], a["q"], a["k"], a["v"], a["out"], self.heads, c.kv, c.dim, c.stride, self.scale,
                      self.nodes, len(self.shapes), c.slot_bytes, a["workspace"], kv_dtype=c.kv_dtype)

    def check(self, out=None):
        got = (self.out if out is None else out).cpu().numpy().reshape(len(self.shapes), self.nodes, self.heads, -1)
        for s, (base, live, parents) in enumerate(self.shapes):
            assert (got[s, live:] == CANARY).all(), "rows behind the live nodes were written"
            if live == 0:
                continue
            want, bound = R.attention(self.caches, s, base, live, parents, self.q[s].reshape(self.nodes, self.heads, -1),
                                      self.heads, self.scale)
            off = np.abs(got[s, :live] - want)
            assert (off <= bound).all(), (s, float(np.nanmax(off / bound)), bool(np.isnan(off).any()))

    def run(self):
        self.call()
        self.check()


@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
@pytest.mark.parametrize("base,nodes", [(0, 1), (0, 5), (1, 1), (1, 21), (37, 4), (58, 6), (59, 6), (63, 1), (64, 22),
                                        (127, 3), (300, 43), (1000, 16)])
def test_one_slot(kv_dtype, base, nodes):
    tree = R.random_tree(np.random.default_rng(base + nodes), nodes)
    Step(base * 1000 + nodes, kv_dtype, [(base, nodes, tree)], nodes).run()


@pytest.mark.parametrize("tree,nodes", [(R.chain, 64), (R.star, 64), (R.chain, 256), (R.star, 256), (R.chain, 65)],
                         ids=["chain 64", "star 64", "chain 256", "star 256", "chain 65"])
def test_wide_and_deep_trees(tree, nodes):
    Step(nodes, 1, [(70, nodes, tree(nodes))], nodes).run()


def test_several_roots_and_a_long_prefix():
    tree = [-1, -1, 0, 1, -1, 2, 3, 4, 4, 0]
    Step(77, 1, [(6000, 10, tree)], 10).run()


@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
@pytest.mark.parametrize("heads,kv,dim", [(6, 1, 256), (8, 1, 256), (4, 4, 256), (15, 5, 256), (8, 2, 64), (3, 1, 32),
                                          (12, 2, 96), (8, 2, 128), (5, 1, 160), (4, 2, 192), (7, 1, 224)])
def test_head_layouts(kv_dtype, heads, kv, dim):
    tree = R.random_tree(np.random.default_rng(dim), 11)
    Step(dim + heads, kv_dtype, [(150, 11, tree)], 11, heads=heads, kv=kv, dim=dim).run()


@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
@pytest.mark.parametrize("dim", [64, 256])
def test_slots_of_unequal_length(kv_dtype, dim):
    rng = np.random.default_rng(5)
    lives = [7, 0, 12, 1, 12, 3]
    bases = [500, 300, 0, 1, 64, 1203]
    shapes = [(b, n, R.random_tree(rng, 12)) for b, n in zip(bases, lives)]
    Step(6, kv_dtype, shapes, 12, heads=6, kv=1 if dim == 256 else 2, dim=dim, pad=48).run()


@pytest.mark.parametrize("slots", [40, 170])
def test_more_slots_than_a_round_of_the_device_holds(slots):
    rng = np.random.default_rng(slots)
    shapes = [(int(rng.integers(0, 200)), int(rng.integers(0, 4)), R.random_tree(rng, 3)) for _ in range(slots)]
    Step(slots, 2, shapes, 3, heads=4, kv=4).run()


def test_no_live_node_at_all():
    Step(1, 1, [(10, 0, []), (0, 0, [])], 4).run()


@pytest.mark.parametrize("kv_dtype,offset,dim", [(0, 4, 256), (0, 8, 64), (1, 2, 256), (1, 6, 64), (2, 2, 256), (2, 4, 96)])
def test_caches_that_are_barely_aligned(kv_dtype, offset, dim):
    shapes = [(200, 9, R.random_tree(np.random.default_rng(8), 9))] * 2
    Step(8, kv_dtype, shapes, 9, heads=4, kv=2, dim=dim, offset=offset, pad=4).run()


def _spoil(step, which, slot, row, value):
    """A cache row's values become `value` (its scales, where it is quantised)."""
    c = step.caches
    raw = c.rows(which, slot)
    if c.kv_dtype == 0:
        raw[:, row] = np.full((c.kv, c.dim), value, dtype=np.float32).view(np.uint8)
    else:
        scale = np.frombuffer(np.float16(value).tobytes(), dtype=np.uint8)
        raw[:, row].reshape(c.kv, -1, R.ROW_BYTES[c.kv_dtype])[:, :, :2] = scale


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_rows_that_are_not_seen_may_hold_anything(dim, kv_dtype, value):
    """Branch 0 -> 1, 0 -> 2: node 2's row and those behind the live nodes are spoilt; nodes 0 and 1 are as before, and what
    sees a spoilt row is not a number."""
    shapes = [(90, 4, [-1, 0, 0, 2])]
    step = Step(3, kv_dtype, shapes, 6, heads=4, kv=2, dim=dim, stride=120)
    for which in (0, 1):
        for row in [92] + list(range(94, 120)):
            _spoil(step, which, 0, row, value)
    step.upload()
    step.call()
    got = step.out.cpu().numpy().reshape(6, 4, dim)
    want, bound = R.attention(step.caches, 0, 90, 2, shapes[0][2], step.q[0].reshape(6, 4, dim), 4, step.scale)
    assert (np.abs(got[:2] - want) <= bound).all()
    assert not np.isfinite(got[2:4]).any()
    assert (got[4:] == CANARY).all()


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("kv_dtype,value", [(0, 3e38), (0, -1e30), (0, 1e7), (1, 65504.0), (1, -900.0), (2, 65504.0)])
def test_rows_that_are_not_seen_may_be_of_any_size(dim, kv_dtype, value):
    """As above, with finite values: nodes 0 and 1 keep all their bits beside a row 2^20 and more times theirs."""
    shapes = [(90, 4, [-1, 0, 0, 2])]
    step = Step(3, kv_dtype, shapes, 6, heads=4, kv=2, dim=dim, stride=120)
    for which in (0, 1):
        for row in [92] + list(range(94, 120)):
            _spoil(step, which, 0, row, value)
    step.upload()
    step.call()
    got = step.out.cpu().numpy().reshape(6, 4, dim)
    want, bound = R.attention(step.caches, 0, 90, 2, shapes[0][2], step.q[0].reshape(6, 4, dim), 4, step.scale)
    assert (np.abs(got[:2] - want) <= bound).all()
    assert (got[4:] == CANARY).all()


@pytest.mark.parametrize("heads,kv,base", [(4, 2, 300), (8, 1, 3000)])
@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
@pytest.mark.parametrize("keys,values", [(24, 0), (0, 24), (20, 20)])
def test_rows_of_very_different_size_side_by_side(heads, kv, base, kv_dtype, keys, values):
    """Rows between their full size and 2^-keys (2^-values) of it, at random along the cache; some are 0."""
    shapes = [(base, 5, R.random_tree(np.random.default_rng(1), 5)), (base // 2, 3, R.chain(3))]
    step = Step(13, kv_dtype, shapes, 5, heads=heads, kv=kv)
    rng = np.random.default_rng(14)
    for s, (b, live, _) in enumerate(shapes):
        for which, spread in ((0, keys), (1, values)):
            size = 2.0 ** (-spread * rng.random((kv, b + live, 1)))
            size[rng.random(size.shape) < 0.05] = 0.0
            step.caches.put(which, s, 0, rng.standard_normal((kv, b + live, 256)) * size)
    step.upload()
    step.run()


def test_f32_rows_of_every_size_side_by_side():
    """Keys of 2^-60 .. 2^60 (their signs make the scores of the large ones -infinity's neighbours), values of 2^-60 .. 2^60."""
    shapes = [(200, 5, R.chain(5))]
    step = Step(15, 0, shapes, 5, heads=4, kv=2)
    rng = np.random.default_rng(16)
    step.q[:] = np.abs(step.q)
    k = -np.abs(rng.standard_normal((2, 205, 256))) * 2.0 ** rng.integers(-60, 61, (2, 205, 1))
    step.caches.put(0, 0, 0, k)
    step.caches.put(1, 0, 0, rng.standard_normal((2, 205, 256)) * 2.0 ** rng.integers(-60, 61, (2, 205, 1)))
    step.upload()
    step.run()


@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
@pytest.mark.parametrize("base", [1500, 5000, 9000])
def test_long_runs_of_one_slot_each(kv_dtype, base):
    """So many slots that a CTA takes 1,500 rows and more in one run: the sums leave the tensor cores' registers on the way."""
    rng = np.random.default_rng(base)
    slots = 40 if base == 1500 else 16
    shapes = [(base + int(rng.integers(0, 70)), 3, R.random_tree(rng, 3)) for _ in range(slots)]
    step = Step(base, kv_dtype, shapes, 3, heads=4, kv=4 if base == 1500 else 1)
    step.run()


def test_long_runs_with_scores_that_fall_and_rise():
    """The largest score comes early, in the middle or late in a long run (what lies in memory outweighs the rest or is outweighed)."""
    slots, base = 40, 2000
    shapes = [(base, 3, R.chain(3))] * slots
    step = Step(17, 1, shapes, 3, heads=4, kv=4)
    rng = np.random.default_rng(18)
    direction = np.sign(rng.standard_normal(256))
    x = np.arange(base + 3)
    for s in range(slots):
        peak = (s + 0.5) / slots * (base + 3)
        size = 12.0 * (1.0 - np.abs(x - peak) / (base + 3))
        step.caches.put(0, s, 0, np.broadcast_to(size[:, None] * direction, (4, base + 3, 256))
                        + 0.3 * rng.standard_normal((4, base + 3, 256)))
    step.q[:] = np.tile(direction, 4) + 0.1 * rng.standard_normal(step.q.shape)
    step.upload()
    step.run()


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("scale", [0.0, -0.05, 3.0])
def test_scales_of_any_sign(dim, scale):
    shapes = [(400, 9, R.random_tree(np.random.default_rng(3), 9))]
    step = Step(19, 1, shapes, 9, heads=4, kv=2, dim=dim)
    step.scale = scale
    step.call()
    got = step.out.cpu().numpy().reshape(9, 4, dim)
    # (the bound's parts that go with the scores take the scale's size)
    want, _ = R.attention(step.caches, 0, 400, 9, shapes[0][2], step.q[0].reshape(9, 4, dim), 4, scale)
    _, bound = R.attention(step.caches, 0, 400, 9, shapes[0][2], np.sign(scale) * step.q[0].reshape(9, 4, dim), 4, abs(scale))
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_queries_that_are_not_finite(dim, value):
    """They are not a number in their own head and node alone."""
    shapes = [(130, 5, R.chain(5))]
    step = Step(20, 1, shapes, 5, heads=4, kv=2, dim=dim)
    clean = step.q.copy()
    step.q.reshape(5, 4, dim)[3, 1, 7] = value
    step.upload()
    step.call()
    got = step.out.cpu().numpy().reshape(5, 4, dim)
    want, bound = R.attention(step.caches, 0, 130, 5, shapes[0][2], clean[0].reshape(5, 4, dim), 4, step.scale)
    others = np.ones((5, 4), dtype=bool)
    others[3, 1] = False
    assert not np.isfinite(got[3, 1]).any()
    assert (np.abs(got - want) <= bound)[others].all()


@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
@pytest.mark.parametrize("k_scale,v_scale", [(1e-3, 1e-4), (30.0, 3000.0), (1.0, 1e-3), (1e-4, 2e4)])
def test_small_and_large_values(kv_dtype, k_scale, v_scale):
    """Keys and values far from 1 (the queries make up for the keys)."""
    shapes = [(333, 9, R.random_tree(np.random.default_rng(2), 9))]
    Step(4, kv_dtype, shapes, 9, q_scale=1.5 / k_scale, k_scale=k_scale, v_scale=v_scale).run()


@pytest.mark.parametrize("k_scale,v_scale", [(1e6, 1e9), (1e-12, 1e-15), (1e15, 1e-20)])
def test_f32_rows_of_any_size(k_scale, v_scale):
    shapes = [(200, 5, R.chain(5))]
    Step(4, 0, shapes, 5, q_scale=1.5 / k_scale, k_scale=k_scale, v_scale=v_scale).run()


@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
def test_scores_that_rise_along_the_cache(kv_dtype):
    """Every tile's largest score exceeds the one before by far, and the last rows carry all the weight."""
    shapes = [(700, 7, R.random_tree(np.random.default_rng(9), 7))]
    step = Step(9, kv_dtype, shapes, 7, heads=6, kv=1)
    rng = np.random.default_rng(10)
    direction = np.sign(rng.standard_normal(256))
    ramp = np.arange(707)[:, None] / 707.0
    step.caches.put(0, 0, 0, (0.5 * rng.standard_normal((707, 256)) + 8.0 * ramp * direction)[None])
    step.q[:] = np.tile(direction, 6) + 0.1 * rng.standard_normal(step.q.shape)
    step.upload()
    step.run()


def test_values_of_very_different_size_along_the_cache():
    """Each slot's f32 value rows grow (or shrink) by a factor of 2^40 along the cache."""
    shapes = [(400, 5, R.chain(5)), (400, 5, R.star(5))]
    step = Step(11, 0, shapes, 5)
    rng = np.random.default_rng(12)
    for s, sign in ((0, 1.0), (1, -1.0)):
        grow = 2.0 ** (sign * 40.0 * np.arange(405) / 405.0)
        step.caches.put(1, s, 0, rng.standard_normal((4, 405, 256)) * grow[None, :, None])
    step.upload()
    step.run()


@pytest.mark.parametrize("dim", [64, 256])
def test_lengths_past_the_cache_count_as_the_cache(dim):
    """(base, end) that reach past the cache: only nodes whose row the cache has are live; negative ones count as 0."""
    tree = R.random_tree(np.random.default_rng(1), 8)
    step = Step(2, 1, [(90, 5, tree), (0, 3, tree), (95, 0, tree), (95, 0, tree)], 8, heads=4, kv=2, dim=dim, stride=95)
    step.parents[:, :] = tree
    step.dparents = _dev(step.parents)
    step.pos = _ints([[90, 98], [-4, 3], [200, 208], [50, 40]])
    step.run()


def test_parents_that_are_no_earlier_nodes():
    """The walk up ends there, whatever stands there; the status names it."""
    tree = [-1, 0, 1, 3, 99, -7, 5, 1 << 30]
    step = Step(21, 1, [(100, 8, tree)], 8)
    step.run()
    _status(41)


@pytest.mark.parametrize("dim", [64, 256])
def test_captured_and_replayed_with_other_lengths_and_trees(dim):
    nodes, rng = 10, np.random.default_rng(31)
    first = Step(30, 1, [(300, 10, R.random_tree(rng, nodes)), (64, 4, R.random_tree(rng, nodes))], nodes, heads=4, kv=2,
                 dim=dim, stride=900)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        first.call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        first.call()
    for shapes in ([(300, 10, R.random_tree(rng, nodes)), (64, 4, R.random_tree(rng, nodes))],
                   [(0, 1, R.chain(nodes)), (890, 10, R.star(nodes))], [(600, 0, []), (700, 3, R.chain(nodes))]):
        other = Step(len(shapes[0][2]) + 40, 1, shapes, nodes, heads=4, kv=2, dim=dim, stride=900)
        for mine, theirs in ((first.pos, other.pos), (first.dparents, other.dparents), (first.dq, other.dq),
                             (first.dk, other.dk), (first.dv, other.dv), (first.out, other.out)):
            mine.copy_(theirs)
        graph.replay()
        torch.cuda.synchronize()
        other.check(first.out)


def test_two_streams_with_workspaces_of_their_own():
    steps = [Step(50 + i, 1 + i, [(2000 - 700 * i, 16, R.random_tree(np.random.default_rng(i), 16))], 16) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(20):
        for step, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                step.call()
    torch.cuda.synchronize()
    for step in steps:
        step.check()


def test_the_same_bits_every_time_whatever_the_workspace_holds():
    step = Step(60, 1, [(3000, 20, R.random_tree(np.random.default_rng(6), 20))], 20)
    step.call()
    first = step.out.clone()
    step.workspace.fill_(1e30)
    step.call()
    assert torch.equal(first, step.out)


@pytest.mark.parametrize("kv_dtype,dim,stride", [(0, 256, 1_200_000), (1, 256, 5_500_000), (2, 64, 40_000_000)],
                         ids=["f32", "q8", "q4"])
def test_offsets_past_32_bits(kv_dtype, dim, stride):
    """The last KV head's rows (or the last rows) begin beyond 4 GB."""
    heads, kv, live = 8, 4, 5
    row = dim * 4 if kv_dtype == 0 else dim // 32 * R.ROW_BYTES[kv_dtype]
    base = stride - 8 if kv_dtype == 0 else 100
    assert (kv_dtype == 0 or 3 * stride * row > 1 << 32) and kv * stride * row > 1 << 32
    rng = np.random.default_rng(70)
    small = R.Caches(kv_dtype, 1, kv, dim, 105)
    small.fill(rng, 0, 105)
    parents = R.chain(live)
    q = rng.standard_normal((live, heads * dim)).astype(np.float32)
    caches = []
    for which in (0, 1):
        rows = _dev(small.rows(which, 0))
        if kv_dtype == 0:
            # (a long prefix is needed to come that far: zero keys and values, which count)
            big = torch.zeros(stride, kv, row, dtype=torch.uint8, device="cuda")
            big[stride - 108:stride - 3] = rows.transpose(0, 1)
        else:
            big = torch.zeros(kv, stride, row, dtype=torch.uint8, device="cuda")
            big[:, :105] = rows
        caches.append(big)
    out = torch.empty(1, live, heads * dim, device="cuda")
    ws = torch.empty(api.attn_tree_workspace_bytes(heads, kv, dim, live, 1), dtype=torch.uint8, device="cuda")
    pos = _ints([[base, base + live]])
    api.attn_tree(pos, _ints([parents]), _dev(q), caches[0], caches[1], out, heads, kv, dim, stride, dim ** -0.5, live, 1, 0, ws,
                  kv_dtype=kv_dtype)
    got = out.cpu().numpy().reshape(live, heads, dim)
    if kv_dtype != 0:
        want, bound = R.attention(small, 0, 100, live, parents, q.reshape(live, heads, dim), heads, dim ** -0.5)
        assert (np.abs(got - want) <= bound).all()
        return
    zeros = stride - 108
    for i in range(live):
        for h in range(heads):
            k, v = (small.values[w][0, h // 2][:100 + i + 1] for w in (0, 1))
            s = dim ** -0.5 * (k @ q[i, h * dim:(h + 1) * dim].astype(np.float64))
            w = np.exp(s)
            want = (w @ v) / (w.sum() + zeros)
            # (1.2 million weights of 1 in the sum: the long sum's part of the bound)
            bound = (2.0 ** -14 + 3 * stride / 16 / 148 * 2.0 ** -23) * (w @ np.abs(v)) / zeros
            assert (np.abs(got[i, h] - want) <= bound).all()


# ---- verification ------------------------------------------------------------------------------------------------

def _softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def _verify(parents, tokens, target, draft, u, lives, bases=None, row_stride=None, offset=0):
    """The device's walk, checked against the reference's for every slot; returns (path, count, next)."""
    slots, nodes, vocab = target.shape
    row_stride = vocab if row_stride is None else row_stride

    def rows(p):
        if p is None:
            return None
        wide = np.full((slots * nodes, row_stride), np.nan, dtype=np.float32)
        wide[:, :vocab] = p.reshape(-1, vocab)
        return _at_offset(wide, offset).view(torch.float32)

    bases = [7] * slots if bases is None else bases
    path = torch.full((slots, nodes), 77, dtype=torch.int32, device="cuda")
    count, following = _ints([55] * slots), _ints([66] * slots)
    api.tree_verify(_ints([[b, b + n] for b, n in zip(bases, lives)]), _ints(parents), _ints(tokens), rows(target), rows(draft),
                    _dev(np.asarray(u, dtype=np.float32)), path, count, following, nodes, slots, vocab, row_stride)
    path, count, following = path.cpu().numpy(), count.cpu().numpy(), following.cpu().numpy()
    for s in range(slots):
        if lives[s] == 0:
            assert (path[s] == 77).all() and count[s] == 55 and following[s] == 66
            continue
        want, token = R.verify(parents[s], tokens[s], target[s], None if draft is None else draft[s],
                               np.asarray(u[s], dtype=np.float32), lives[s])
        assert list(path[s]) == want + [-1] * (nodes - len(want)), s
        assert count[s] == len(want) and following[s] == token, (s, following[s], token)
    return path, count, following


def _drafted(rng, slots, nodes, vocab, width, near=0.8, peak=3.0):
    """Trees whose tokens were drawn from the parents' draft rows."""
    logits = peak * rng.standard_normal((slots, nodes, vocab))
    target, draft = _softmax(logits), _softmax(logits + near * rng.standard_normal(logits.shape))
    parents = [R.random_tree(rng, nodes, width) for _ in range(slots)]
    tokens = np.zeros((slots, nodes), dtype=np.int32)
    for s in range(slots):
        for i in range(1, nodes):
            c = np.cumsum(draft[s, parents[s][i]].astype(np.float64))
            tokens[s, i] = min(vocab - 1, int(np.searchsorted(c, rng.random() * c[-1])))
    u = rng.random((slots, nodes)).astype(np.float32)
    return parents, tokens.tolist(), target, draft, u


@pytest.mark.parametrize("looked_up", [False, True], ids=["drawn", "looked up"])
@pytest.mark.parametrize("slots,nodes,vocab,width", [(1, 1, 100, 1), (1, 2, 1, 1), (3, 8, 5, 1), (4, 16, 31, 3), (2, 6, 32, 6),
                                                     (2, 6, 33, 6), (3, 12, 1000, 3), (2, 9, 16383, 8), (2, 5, 50257, 3),
                                                     (1, 4, 151936, 3), (1, 3, 300001, 2)])
def test_walks(looked_up, slots, nodes, vocab, width):
    rng = np.random.default_rng(vocab + nodes)
    for _ in range(3):
        parents, tokens, target, draft, u = _drafted(rng, slots, nodes, vocab, width)
        lives = [int(rng.integers(0 if slots > 1 else 1, nodes + 1)) for _ in range(slots)]
        _verify(parents, tokens, target, None if looked_up else draft, u, lives)


@pytest.mark.parametrize("looked_up", [False, True], ids=["drawn", "looked up"])
def test_the_widest_and_the_deepest_tree(looked_up):
    rng = np.random.default_rng(3)
    slots, nodes, vocab = 2, 256, 40
    _, _, target, draft, u = _drafted(rng, slots, nodes, vocab, 4, near=2.0)
    parents = [R.star(nodes), R.chain(nodes)]
    tokens = rng.integers(0, vocab, (slots, nodes)).tolist()
    # the chain's tokens are the target's: most are kept
    tokens[1] = [0] + [int(target[1, i].argmax()) for i in range(nodes - 1)]
    u[1, 1:] *= 0.5
    _verify(parents, tokens, target, None if looked_up else draft, u, [nodes, nodes])


@pytest.mark.parametrize("row_stride,offset", [(1003, 0), (1004, 0), (1001, 4), (1008, 16), (1008, 8)])
def test_rows_apart_and_barely_aligned(row_stride, offset):
    rng = np.random.default_rng(row_stride)
    parents, tokens, target, draft, u = _drafted(rng, 3, 7, 1001, 3)
    _verify(parents, tokens, target, draft, u, [7, 7, 7], row_stride=row_stride, offset=offset)


@pytest.mark.parametrize("looked_up", [False, True], ids=["drawn", "looked up"])
@pytest.mark.parametrize("u0", [0.0, 2.0 ** -24, 0.5, 1.0 - 2.0 ** -24])
def test_random_numbers_at_the_ends(looked_up, u0):
    rng = np.random.default_rng(9)
    for u_rest in (0.0, 1.0 - 2.0 ** -24):
        parents, tokens, target, draft, u = _drafted(rng, 4, 6, 3000, 4)
        target[:, :, :5] = 0.0
        target[:, :, -700:] = 0.0   # the last token with mass lies inside
        u[:, 1:], u[:, 0] = u_rest, u0
        _verify(parents, tokens, target, None if looked_up else draft, u, [6] * 4)


@pytest.mark.parametrize("looked_up", [False, True], ids=["drawn", "looked up"])
def test_rows_without_mass_and_what_is_no_probability(looked_up):
    rng = np.random.default_rng(10)
    parents, tokens, target, draft, u = _drafted(rng, 5, 6, 500, 3)
    target[0] = 0.0
    target[1, :, ::3] = np.nan
    target[2, :, 1::3] = -1.0
    target[3, :, 2::7] = np.inf
    draft[1, :, ::2] = np.nan
    draft[4, :, ::5] = np.inf
    _, _, following = _verify(parents, tokens, target, None if looked_up else draft, u, [6] * 5)
    assert following[0] == -1


def test_rejections_that_leave_nothing():
    """A draft that exceeds the target everywhere: the target itself stays, for the later children and for the next token."""
    target = np.zeros((1, 4, 64), dtype=np.float32)
    target[0, :, 8:16] = 0.125
    draft = np.full((1, 4, 64), 0.9, dtype=np.float32)
    for u in ([0.3, 0.9, 0.9, 0.9], [0.3, 0.9, 0.9, 0.1]):
        _verify([R.star(4)], [[0, 9, 9, 10]], target, draft, np.array([u], dtype=np.float32), [4])


@pytest.mark.parametrize("slots,vocab", [(1, 151936), (3, 50257), (12, 4099), (40, 1000)])
@pytest.mark.parametrize("looked_up", [False, True], ids=["drawn", "looked up"])
def test_many_rejections_in_a_row(looked_up, slots, vocab):
    """Every child of a wide tree is refused (its token's probability is next to nothing, or taken before)."""
    rng = np.random.default_rng(vocab)
    nodes = 12
    _, _, target, draft, u = _drafted(rng, slots, nodes, vocab, 3, near=1.5)
    parents = [R.star(nodes) if s % 2 == 0 else [-1] + [0] * 5 + [1] * (nodes - 6) for s in range(slots)]
    # the root's tokens: some of the most probable ones, some twice
    tokens = []
    for s in range(slots):
        order = np.argsort(-target[s, 0])
        tokens.append([0] + [int(order[j % 7]) for j in range(nodes - 1)])
    u[:, 1:] = 1.0 - 2.0 ** -24
    _verify(parents, tokens, target, None if looked_up else draft, u, [nodes] * slots)


def test_rejected_tokens_that_hold_nearly_all():
    """Looked-up tokens take all but some 2^-20 of the mass away: what is left is summed anew, not taken off."""
    nodes, vocab = 6, 5000
    target = np.full((1, nodes, vocab), 2.0 ** -33, dtype=np.float32)
    target[0, :, 100:105] = [0.5, 0.25, 0.125, 0.0625, 0.0625]
    tokens = [[0, 100, 101, 102, 103, 104]]
    for u0 in (0.0, 0.3, 0.999):
        u = np.array([[u0] + [1.0 - 2.0 ** -24] * (nodes - 1)], dtype=np.float32)
        _, count, _ = _verify([R.star(nodes)], tokens, target, None, u, [nodes])


def test_looked_up_children_that_hold_all_of_the_mass():
    """Rejections without draft rows down to nothing: the last token with mass stays, for later siblings and the next token."""
    nodes, vocab = 8, 200
    for mass, tokens in (([(5, 0.5), (9, 0.5)], [0, 5, 9, 7, 9, 5, 9, 3]), ([(5, 1.0)], [0, 5, 7, 5, 8, 5, 5, 5]),
                         ([(5, 1.0)], [0, 7, 8, 5, 5, 7, 5, 9]), ([], [0, 5, 7, 5, 8, 5, 5, 5]),
                         ([(5, 0.25), (9, 0.5), (199, 0.25)], [0, 9, 9, 199, 9, 5, 5, 9])):
        target = np.zeros((1, nodes, vocab), dtype=np.float32)
        for x, m in mass:
            target[0, :, x] = m
        # (no random number of 1: a first token that has all of the mass is kept; larger ones make the walk refuse it)
        for u in (0.5, 0.99, 1.0, 4.0):
            for parents in (R.star(nodes), [-1, 0, 0, 0, 3, 3, 0, 6]):
                for u0 in (0.0, 0.6):
                    _verify([parents], [tokens], target, None, np.array([[u0] + [u] * (nodes - 1)], dtype=np.float32), [nodes])


def test_siblings_with_the_same_token():
    rng = np.random.default_rng(12)
    for _ in range(6):
        parents, tokens, target, draft, u = _drafted(rng, 3, 7, 9, 7)
        parents, tokens = [R.star(7)] * 3, [[0, 4, 4, 4, 5, 5, 4]] * 3
        u[:, 1:] = 0.5 + 0.5 * u[:, 1:]
        _verify(parents, tokens, target, draft, u, [7] * 3)
        _verify(parents, tokens, target, None, u, [7] * 3)


def test_children_that_are_never_kept():
    """Parents that are no earlier node and tokens outside the vocabulary; the status names them."""
    rng = np.random.default_rng(13)
    parents, tokens, target, draft, u = _drafted(rng, 2, 8, 100, 2)
    u[:, 1:] = 0.0
    parents = [[-1, 0, 0, 2, 7, 4, -5, 6], [-1, -1, 0, 2, 3, 1 << 30, 4, 6]]
    tokens[0][2], tokens[1][4] = 100, -1
    _verify(parents, tokens, target, draft, u, [8, 8])
    _status(41)


def test_many_slots_emit_the_targets_distribution():
    """60,000 slots with one row of eight tokens: the token that comes first has the target's probability, within five
    standard deviations of each count."""
    rng = np.random.default_rng(14)
    slots, nodes, vocab = 60_000, 4, 8
    p, q = _softmax(1.5 * rng.standard_normal(vocab)), _softmax(1.5 * rng.standard_normal(vocab))
    tokens = rng.choice(vocab, (slots, nodes), p=q.astype(np.float64) / q.astype(np.float64).sum()).astype(np.int32)
    u = rng.random((slots, nodes)).astype(np.float32)
    target = _dev(np.tile(p, (slots, nodes, 1)))
    draft = _dev(np.tile(q, (slots, nodes, 1)))
    path = torch.empty(slots, nodes, dtype=torch.int32, device="cuda")
    count, following = _ints([0] * slots), _ints([0] * slots)
    api.tree_verify(_ints([[0, nodes]] * slots), _ints([R.star(nodes)] * slots), _dev(tokens), target, draft, _dev(u), path,
                    count, following, nodes, slots, vocab)
    path, count, following = path.cpu().numpy(), count.cpu().numpy(), following.cpu().numpy()
    emitted = np.where(count > 1, tokens[np.arange(slots), np.maximum(path[:, 1], 0)], following)
    got = np.bincount(emitted, minlength=vocab)
    assert (np.abs(got - slots * p) <= 5 * np.sqrt(slots * p * (1 - p))).all()


def test_verification_captured_and_replayed():
    rng = np.random.default_rng(15)
    sets = [_drafted(rng, 3, 6, 2000, 3) for _ in range(3)]

    def tensors(x):
        parents, tokens, target, draft, u = x
        return [_ints(parents), _ints(tokens), _dev(target), _dev(draft), _dev(u)]

    mine = tensors(sets[0])
    pos = _ints([[5, 11]] * 3)
    path, count, following = torch.zeros(3, 6, dtype=torch.int32, device="cuda"), _ints([0] * 3), _ints([0] * 3)

    def call():
        api.tree_verify(pos, *mine, path, count, following, 6, 3, 2000)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for x in sets:
        for a, b in zip(mine, tensors(x)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for s in range(3):
            want, token = R.verify(x[0][s], x[1][s], x[2][s], x[3][s], x[4][s], 6)
            assert path[s].tolist() == want + [-1] * (6 - len(want)) and following[s] == token and count[s] == len(want)


# ---- the kept path -----------------------------------------------------------------------------------------------

class Rows:
    """Caches of random bytes with paths, on the device."""

    def __init__(self, seed, kv_dtype, shapes, nodes, paths, layers=2, kv=4, dim=256, stride=None, offset=0, pad=0):
        rng = np.random.default_rng(seed)
        self.nodes, self.paths, self.bases = nodes, paths, [b for b, _ in shapes]
        stride = max(b + n for b, n in shapes) + 5 if stride is None else stride
        c = R.Caches(kv_dtype, len(shapes), kv, dim, stride, pad=pad)
        self.caches, self.layers = c, layers
        self.host = [rng.integers(0, 256, c.slot_bytes * len(shapes), dtype=np.uint8) for _ in range(2 * layers)]
        self.device = [_at_offset(h, offset) for h in self.host]
        self.pos = _ints([[b, b + n] for b, n in shapes])
        self.path = _ints([p + [99] * (nodes - len(p)) for p in paths])
        self.count = _ints([len(p) for p in paths])

    def call(self):
        c = self.caches
        api.kv_path_keep(self.pos, self.path, self.count, self.device[:self.layers], self.device[self.layers:], c.kv, c.dim,
                         c.stride, self.nodes, c.slots, c.slot_bytes, kv_dtype=c.kv_dtype)

    def check(self, moved=None):
        """Every byte of every cache; `moved`: the slots whose rows move (all)."""
        c = self.caches
        for host, device in zip(self.host, self.device):
            c.bytes = [host.copy()]
            for s, path in enumerate(self.paths):
                if moved is not None and s not in moved:
                    continue
                old, rows = c.rows(0, s).copy(), c.rows(0, s)
                for i, node in enumerate(path):
                    rows[:, self.bases[s] + i] = old[:, self.bases[s] + node]
            assert np.array_equal(c.bytes[0], device.cpu().numpy())


@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
@pytest.mark.parametrize("kv,dim,offset", [(4, 256, 0), (1, 256, 4), (2, 64, 0), (3, 32, 8), (2, 96, 0), (5, 224, 12)])
def test_paths_move(kv_dtype, kv, dim, offset):
    shapes = [(100, 16), (0, 9), (37, 16), (5, 1), (60, 0), (8, 16)]
    paths = [[0, 2, 5, 6, 11, 15], [0, 1, 2, 3], [0, 15], [0], [], list(range(1, 16))]
    rows = Rows(dim + kv, kv_dtype, shapes, 16, paths, kv=kv, dim=dim, offset=offset, pad=36)
    rows.call()
    rows.check()


@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
def test_the_longest_paths(kv_dtype):
    rng = np.random.default_rng(1)
    some = sorted(rng.choice(256, 200, replace=False).tolist())
    rows = Rows(2, kv_dtype, [(40, 256), (0, 256), (3, 256)], 256, [some, list(range(256)), list(range(1, 256))], layers=1)
    rows.call()
    rows.check()


@pytest.mark.parametrize("layers", [1, 64, 65, 130])
def test_numbers_of_layers(layers):
    rows = Rows(layers, 1, [(10, 6)], 6, [[0, 3, 5]], layers=layers, kv=1, dim=64)
    rows.call()
    rows.check()


@pytest.mark.parametrize("path", [[0, 2, 2], [2, 1], [0, 8], [-1, 2], [0, 3, 6], [3, 1 << 30], [1, -(1 << 31)]], ids=str)
def test_paths_that_do_not_ascend_in_their_tree_move_nothing(path):
    """(six live nodes of eight)"""
    rows = Rows(3, 1, [(10, 6), (4, 6)], 8, [path, [0, 2, 4]], kv=2, dim=64)
    rows.call()
    _status(42)
    rows.check(moved=[1])


@pytest.mark.parametrize("count", [-1, 7, 8, 1 << 30])
def test_counts_past_the_tree_move_nothing(count):
    rows = Rows(4, 2, [(10, 6), (4, 6)], 8, [[0, 2, 3], [0, 2, 4]], kv=2, dim=64)
    rows.count = _ints([count, 3])
    rows.call()
    _status(42)
    rows.check(moved=[1])


def test_rows_of_a_tree_past_the_cache():
    """The cache ends inside the tree: its last nodes are not live."""
    rows = Rows(5, 1, [(10, 6), (12, 3)], 8, [[0, 2, 5], [1, 2]], kv=2, dim=64, stride=15)
    rows.pos = _ints([[10, 16], [12, 18]])
    rows.call()
    _status(42)
    rows.check(moved=[1])


# ---- the step ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv_dtype", [0, 1, 2], ids=["f32", "q8", "q4"])
def test_a_step_of_speculation(kv_dtype):
    """Append the drafted rows, attend, verify, keep; then every cache is what appending the kept rows alone makes it, and the
    last kept node's attention is what one decode column over that cache gives."""
    rng = np.random.default_rng(80 + kv_dtype)
    heads, kv, dim, nodes, base, layers, vocab = 24, 4, 256, 12, 500, 3, 700
    stride = 600
    parents, tokens, target, draft, u = _drafted(rng, 1, nodes, vocab, 3, near=0.2)
    u[:, 1:] *= 0.6
    caches = []
    for _ in range(layers):
        c = R.Caches(kv_dtype, 1, kv, dim, stride, fill=0)
        c.fill(rng, 0, base)
        caches.append([_dev(b) for b in c.bytes])
    fresh = [[t.clone() for t in pair] for pair in caches]
    k, v = (torch.from_numpy(rng.standard_normal((layers, nodes, kv * dim)).astype(np.float32)).cuda() for _ in range(2))
    q = torch.from_numpy((1.5 * rng.standard_normal((layers, 1, nodes, heads * dim))).astype(np.float32)).cuda()
    out = torch.zeros_like(q)
    ws = torch.empty(api.attn_tree_workspace_bytes(heads, kv, dim, nodes, 1), dtype=torch.uint8, device="cuda")
    pos, dparents = _ints([[base, base + nodes]]), _ints(parents)

    def append(pair, rows_k, rows_v, n):
        if kv_dtype == 0:
            api.kv_append_chunk_f32(pair[0].view(torch.float32), pair[1].view(torch.float32), rows_k, rows_v, base, kv * dim, n)
        else:
            api.kv_encode_bulk(rows_k, rows_v, *pair, kv, dim, stride, base, 0, n, dtype=kv_dtype - 1)

    for layer in range(layers):
        append(caches[layer], k[layer], v[layer], nodes)
        api.attn_tree(pos, dparents, q[layer], *caches[layer], out[layer], heads, kv, dim, stride, dim ** -0.5, nodes, 1, 0, ws,
                      kv_dtype=kv_dtype)
    path, count, following = torch.zeros(1, nodes, dtype=torch.int32, device="cuda"), _ints([0]), _ints([0])
    api.tree_verify(pos, dparents, _ints(tokens), _dev(target), _dev(draft), _dev(u), path, count, following, nodes, 1, vocab)
    api.kv_path_keep(pos, path, count, [c[0] for c in caches], [c[1] for c in caches], kv, dim, stride, nodes, 1, 0,
                     kv_dtype=kv_dtype)
    kept, token = R.verify(parents[0], tokens[0], target[0], draft[0], u[0], nodes)
    n = int(count[0])
    assert n == len(kept) > 1 and path[0, :n].tolist() == kept and int(following[0]) == token
    index = torch.tensor(kept, device="cuda")
    for layer in range(layers):
        append(fresh[layer], k[layer][index].contiguous(), v[layer][index].contiguous(), n)
        live = base + n
        for a, b in zip(caches[layer], fresh[layer]):
            row = a.numel() // (kv * stride)
            shape = (stride, kv, row) if kv_dtype == 0 else (kv, stride, row)
            cut = (lambda t: t.view(shape)[:live]) if kv_dtype == 0 else (lambda t: t.view(shape)[:, :live])
            assert torch.equal(cut(a), cut(b))
        # one more decode column at the last kept node
        last = q[layer, 0, kept[-1]].contiguous()
        one = torch.empty(heads * dim, device="cuda")
        if kv_dtype == 0:
            splits = api.cols_splits(stride)
            api.attn_decode_cols_f32(last, caches[layer][0], caches[layer][1], torch.empty(heads * splits * dim, device="cuda"),
                                     torch.empty(heads * splits * 2, device="cuda"), one, heads, kv, dim, stride, live - 1, 1)
        else:
            splits = api.decode_splits(live)
            api.attn_decode_kv(_ints([live - 1, live, 0, 0, 0, 0, 0, 0]), last, *caches[layer],
                               torch.empty(heads * splits * dim, device="cuda"), torch.empty(heads * splits * 2, device="cuda"),
                               one, heads, kv, dim, stride, dim ** -0.5, splits, selector=kv_dtype - 1)
        # both are within the decode entries' bar of the definition
        assert float((one - out[layer, 0, kept[-1]]).abs().max()) <= 4e-5
