"""What the entries of tree speculation refuse, and the walk's rule on small numbers. No GPU: a refused call ends before
anything is launched."""
import ctypes as C

import numpy as np
import pytest

from hipml_b200 import _lib, api
from tests import tree_reference as R


class _At:
    def __init__(self, address=4096):
        self.address = address

    def data_ptr(self):
        return self.address

    def numel(self):
        return 1 << 40

    def element_size(self):
        return 1


T = _At()


class _Calls:
    """The call module over ctypes: the native one asks torch for its stream, which needs a device."""

    def __getattr__(self, name):
        def call(*args):
            if name == "kv_path_keep":
                kv_dtype, pos, path, count, k, v, *rest = args
                n = max(len(k), len(v))
                tables = [(C.c_void_p * max(n, 1))(*[x.data_ptr() for x in c]) for c in (k, v)]
                args = [kv_dtype, pos, path, count, *tables, n, *rest]
            args = [x.data_ptr() if hasattr(x, "data_ptr") else x for x in args]
            return getattr(_lib.load(), "hipml_" + name)(None, *args)
        return call


@pytest.fixture(autouse=True)
def calls(monkeypatch):
    monkeypatch.setattr(api, "_c", _Calls())


def _attn(pos=T, parents=T, q=T, k=T, v=T, out=T, heads=24, kv=4, dim=256, stride=100, nodes=8, slots=1, slot_bytes=0,
          workspace=T, kv_dtype=1):
    api.attn_tree(pos, parents, q, k, v, out, heads, kv, dim, stride, 0.0625, nodes, slots, slot_bytes, workspace,
                  kv_dtype=kv_dtype)


class _Small(_At):
    def numel(self):
        return 1000


@pytest.mark.parametrize("args,text", [
    (dict(kv_dtype=3), "unknown KV dtype 3"), (dict(kv_dtype=-1), "unknown KV dtype -1"),
    (dict(heads=25), "not a multiple"), (dict(heads=0), "n_heads 0"), (dict(heads=36), "GQA group 9"), (dict(kv=0), "n_kv 0"),
    (dict(dim=48), "head_dim 48"), (dict(dim=288), "head_dim 288"), (dict(stride=0), "stride 0"),
    (dict(nodes=0), "tree of 0 nodes"), (dict(nodes=257), "tree of 257 nodes"), (dict(slots=0), "slots 0"),
    (dict(slots=65536), "slots 65536"),
    (dict(slots=2, slot_bytes=4 * 100 * 272 - 2), "bytes a slot"), (dict(slots=2, slot_bytes=4 * 100 * 272 + 1), "bytes a slot"),
    (dict(pos=None), "missing"), (dict(parents=None), "missing"), (dict(q=None), "missing"), (dict(k=None), "missing"),
    (dict(v=None), "missing"), (dict(out=None), "missing"), (dict(q=_At(4100)), "16-byte"), (dict(out=_At(4104)), "16-byte"),
    (dict(k=_At(4097)), "2-byte"), (dict(kv_dtype=0, v=_At(4098)), "4-byte"),
], ids=str)
def test_attention_refuses(args, text):
    with pytest.raises(_lib.HipmlError, match=text) as e:
        _attn(**args)
    assert e.value.code == _lib.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("workspace,text", [(None, "needed"), (_Small(), "1000 bytes given"), (_At(4100), "16-byte")], ids=str)
def test_attention_wants_its_workspace(workspace, text):
    with pytest.raises(_lib.HipmlError, match=text) as e:
        _attn(workspace=workspace)
    assert e.value.code == _lib.ERR_WORKSPACE


def test_workspace_grows_with_what_is_asked_and_is_0_for_what_is_refused():
    at = api.attn_tree_workspace_bytes
    assert 0 < at(24, 4, 256, 1, 1) <= at(24, 4, 256, 64, 1) <= at(24, 4, 256, 64, 64) <= at(24, 4, 256, 256, 64)
    assert at(24, 4, 256, 0, 1) == at(24, 4, 256, 257, 1) == at(25, 4, 256, 8, 1) == at(24, 4, 250, 8, 1) == 0
    assert at(24, 0, 256, 8, 1) == at(0, 4, 256, 8, 1) == at(24, 4, 256, 8, 0) == 0


def _verify(pos=T, parents=T, tokens=T, target=T, draft=None, uniform=T, path=T, count=T, following=T, nodes=8, slots=1,
            vocab=100, row_stride=None):
    api.tree_verify(pos, parents, tokens, target, draft, uniform, path, count, following, nodes, slots, vocab, row_stride)


@pytest.mark.parametrize("args,text", [
    (dict(nodes=0), "tree of 0"), (dict(nodes=300), "tree of 300"), (dict(slots=0), "slots 0"), (dict(vocab=0), "vocabulary of 0"),
    (dict(vocab=(1 << 20) + 1), "vocabulary of 1048577"), (dict(row_stride=99), "rows of 99"),
    *[({k: None}, "missing") for k in ("pos", "parents", "tokens", "target", "uniform", "path", "count", "following")],
], ids=str)
def test_verification_refuses(args, text):
    with pytest.raises(_lib.HipmlError, match=text) as e:
        _verify(**args)
    assert e.value.code == _lib.ERR_INVALID_ARGUMENT


def _keep(pos=T, path=T, count=T, k=(T,), v=(_At(8192),), kv=4, dim=256, stride=100, nodes=8, slots=1, slot_bytes=0,
          kv_dtype=1):
    api.kv_path_keep(pos, path, count, k, v, kv, dim, stride, nodes, slots, slot_bytes, kv_dtype=kv_dtype)


@pytest.mark.parametrize("args,text", [
    (dict(kv_dtype=3), "unknown KV dtype"), (dict(kv=0), "n_kv 0"), (dict(dim=40), "head_dim 40"), (dict(stride=0), "stride 0"),
    (dict(nodes=0), "tree of 0"), (dict(slots=0), "slots 0"), (dict(slots=2, slot_bytes=100), "bytes a slot"),
    (dict(pos=None), "missing"), (dict(path=None), "missing"), (dict(count=None), "missing"),
    (dict(k=(T, _At(1 << 20))), "cache 3 is missing"), (dict(k=(_At(4097),)), "2-byte"),
    (dict(kv_dtype=0, k=(_At(4098),)), "4-byte"), (dict(k=(T,), v=(T,)), "caches 0 and 1 are the same"),
    (dict(k=(T, _At(8)), v=(_At(16), _At(8))), "caches 1 and 3 are the same"),
], ids=str)
def test_path_refuses(args, text):
    with pytest.raises(_lib.HipmlError, match=text) as e:
        _keep(**args)
    assert e.value.code == _lib.ERR_INVALID_ARGUMENT


def test_no_layers_is_no_work():
    _keep(k=(), v=())
    assert _lib.load().hipml_kv_path_keep(None, 1, None, None, None, None, None, -1, 4, 256, 8, 8, 1, 0) \
        == _lib.ERR_INVALID_ARGUMENT


def test_the_native_view_takes_sequences_of_caches(monkeypatch):
    monkeypatch.setattr(api, "_c", _lib.calls())
    asked = []

    class One:
        def __init__(self, at):
            self.at = at

        def data_ptr(self):
            asked.append(self.at)
            return self.at

    with pytest.raises(TypeError):
        _keep(k=3)
    with pytest.raises(TypeError):   # of the last argument: all before it were taken
        _keep(k=[One(64), One(128)], v=(One(192), One(256)), slot_bytes="x")
    assert asked == [64, 128, 192, 256]


def test_the_rule_emits_the_targets_distribution():
    """The reference walk itself: over a fine grid of random numbers the first token that a tree of two children and a root
    emits (a kept child's token, or the drawn one) has the target's probabilities, to within the grid."""
    p = np.array([0.5, 0.2, 0.2, 0.1])
    q = np.array([0.1, 0.6, 0.2, 0.1])
    n, got = 24, np.zeros(4)
    grid = (np.arange(n) + 0.5) / n
    target, draft = np.tile(p, (3, 1)), np.tile(q, (3, 1))
    for a in range(4):
        for b in range(4):
            for u1 in grid:
                for u2 in grid:
                    # (the drawn token's number only matters where both are rejected: take its mean)
                    path, _ = R.verify(R.star(3), [0, a, b], target, draft, [0.5, u1, u2], 3)
                    w = q[a] * q[b] / n / n
                    if len(path) > 1:
                        got[(a, b)[path[1] - 1]] += w
                    else:
                        for u0 in grid:
                            got[R.verify(R.star(3), [0, a, b], target, draft, [u0, u1, u2], 3)[1]] += w / n
    # each of the three numbers moves a share of at most one cell of the grid
    assert np.abs(got - p).max() <= 3.0 / n


@pytest.mark.parametrize("stride", [0, -5])
def test_verification_refuses_a_cache_without_rows(stride):
    with pytest.raises(_lib.HipmlError, match=f"stride {stride} must be positive"):
        api.tree_verify(T, T, T, T, None, T, T, T, T, 8, 1, 100, stride=stride)
    with pytest.raises(_lib.HipmlError, match="vocabulary of 0"):   # the bound changes nothing of the other refusals
        api.tree_verify(T, T, T, T, None, T, T, T, T, 8, 1, 0, stride=100)


def test_attention_refuses_more_pairs_of_tiles_than_the_plan_counts():
    """64 row tiles (256 nodes of eight heads) over 2^25 key tiles are 2^31 pairs: two slots of them do not fit 32 bits."""
    rows = (1 << 31) - 1
    with pytest.raises(_lib.HipmlError, match="256 nodes over 2 slots of 2147483647 rows are too many") as e:
        _attn(heads=8, kv=1, dim=32, nodes=256, slots=2, stride=rows, slot_bytes=rows * 18, kv_dtype=2)
    assert e.value.code == _lib.ERR_INVALID_ARGUMENT
    # (one slot, or 128 nodes, are as many as it counts: what is missing there is the workspace)
    for few in (dict(slots=1), dict(nodes=127)):
        with pytest.raises(_lib.HipmlError, match="needed"):
            _attn(**{**dict(heads=8, kv=1, dim=32, nodes=256, slots=2, stride=rows, slot_bytes=rows * 18, kv_dtype=2,
                            workspace=None), **few})
