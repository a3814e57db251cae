"""CPU tests of a step of drafted tokens over a paged cache: what the entry points refuse (their checks alone, no GPU)."""
import pytest
import torch

from cuvs_b200 import _lib as L
from cuvs_b200 import kv_cache
from test_kv_cache import DEVICE, Described

H, I, F, W = torch.float16, torch.int32, torch.float32, torch.uint32
A, D, T, K, P = kv_cache._APPEND_TURNED, kv_cache._DRAFT_TREE, kv_cache._ATTEND_TREE, kv_cache._KEEP_PATH, kv_cache._COPY_PAGES
OPS = [A, D, T, K, P]
TREE = (0, kv_cache._bits(0.125), kv_cache._bits(0.0))


def described(op):
    """The tensors of a good call, by name, and its scalars."""
    cache = {"keys": Described(H, (9, 16, 4, 64)), "values": Described(H, (9, 16, 4, 64))}
    if op == A:
        return {**cache, "new_keys": Described(H, (5, 4, 64)), "new_values": Described(H, (5, 4, 64)), "pages": Described(I, (3, 7)),
                "positions": Described(I, (5,)), "sequences": Described(I, (5,)), "queries": Described(H, (5, 8, 64)),
                "frequencies": Described(torch.float64, (32,)), "slots": Described(torch.int64, (5,)), "rotated": Described(H, (5, 8, 64)),
                "turns": Described(I, (5, 3)), "axes": Described(I, (32,))}, (0,)
    if op == D:
        return {"parents": Described(I, (3, 40)), "lengths": Described(I, (3,)), "mask": Described(W, (3, 40, 2)),
                "positions": Described(I, (3, 40))}, ()
    if op == T:
        return {**cache, "queries": Described(H, (3, 40, 8, 64)), "pages": Described(I, (3, 7)), "lengths": Described(I, (3,)),
                "positions": Described(I, (3, 40)), "mask": Described(W, (3, 40, 2)), "slopes": Described(F, (8,)),
                "filter": Described(W, (5,)), "out": Described(H, (3, 40, 8, 64)), "lse": Described(F, (3, 40, 8)),
                "workspace": Described(torch.uint8, (1 << 20,))}, TREE
    if op == K:
        return {**cache, "pages": Described(I, (3, 7)), "lengths": Described(I, (3,)), "paths": Described(I, (3, 6)),
                "kept": Described(I, (3,), address=1 << 41)}, ()
    return {**cache, "sources": Described(I, (4,)), "targets": Described(I, (4,))}, ()


OPTIONAL = {A: {"sequences", "axes"}, T: {"slopes", "filter", "workspace"}}


def check(op, changes=None, scalars=None):
    tensors, usual = described(op)
    tensors.update(changes or {})
    L.check(L.load().cuvsB200KvCacheCheck(DEVICE, op, *kv_cache._words(tensors.values(), usual if scalars is None else scalars)))


@pytest.mark.parametrize("op", OPS)
def test_good_calls_pass_and_calls_without_a_tensor_do_not(op):
    check(op)
    for name in described(op)[0]:
        if name in OPTIONAL.get(op, ()):
            if name not in ("sequences", "axes"):
                check(op, {name: None})
        else:
            with pytest.raises(L.CuvsError, match="null tensor|together|go with frequencies"):
                check(op, {name: None})


@pytest.mark.parametrize("op", OPS)
def test_tensors_of_another_place_or_rank_are_refused(op):
    for name, t in described(op)[0].items():
        with pytest.raises(L.CuvsError, match="expected a CUDA tensor"):
            check(op, {name: Described(t.dtype, t.shape, device=-1)})
        with pytest.raises(L.CuvsError, match="but the handle is for device 3"):
            check(op, {name: Described(t.dtype, t.shape, device=1)})
        if len(t.shape) < 4:
            with pytest.raises(L.CuvsError, match="dimensions"):
                check(op, {name: Described(t.dtype, t.shape + (1,))})


@pytest.mark.parametrize("op,name,tensor,message", [
    # element types
    (A, "turns", Described(torch.int64, (5, 3)), "expected int32"),
    (A, "axes", Described(torch.int64, (32,)), "expected int32"),
    (D, "parents", Described(torch.int64, (3, 40)), "expected int32"),
    (D, "mask", Described(I, (3, 40, 2)), "expected uint32"),
    (D, "positions", Described(F, (3, 40)), "expected int32"),
    (T, "queries", Described(F, (3, 40, 8, 64)), "element type"),
    (T, "mask", Described(I, (3, 40, 2)), "expected uint32"),
    (T, "slopes", Described(H, (8,)), "expected float32"),
    (T, "lse", Described(H, (3, 40, 8)), "expected float32"),
    (T, "positions", Described(torch.int64, (3, 40)), "expected int32"),
    (K, "paths", Described(torch.int64, (3, 6)), "expected int32"),
    (K, "kept", Described(torch.int64, (3,)), "expected int32"),
    (K, "keys", Described(torch.float64, (9, 16, 4, 64)), "unsupported element type"),
    (P, "sources", Described(torch.int64, (4,)), "expected int32"),
    # shapes that do not go together
    (A, "turns", Described(I, (4, 3)), "one row for each token"),
    (A, "turns", Described(I, (5, 0)), "1 to 65535 axes"),
    (A, "axes", Described(I, (31,)), "one for each pair"),
    (D, "parents", Described(I, (3, 0)), "1 to 1024 drafted"),
    (D, "parents", Described(I, (3, 1025)), "1 to 1024 drafted"),
    (D, "lengths", Described(I, (2,)), "one for each sequence"),
    (D, "mask", Described(W, (3, 40, 3)), "mask: expected shape"),
    (D, "positions", Described(I, (3, 41)), "positions: expected shape"),
    (T, "queries", Described(H, (3, 40, 6, 64)), "no multiple"),
    (T, "queries", Described(H, (3, 40, 0, 64)), "no multiple"),
    (T, "queries", Described(H, (3, 0, 8, 64)), "1 to 1024 drafted"),
    (T, "queries", Described(H, (3, 40, 8, 72)), "rows of 64 elements"),
    (T, "pages", Described(I, (2, 7)), "a row for each"),
    (T, "lengths", Described(I, (4,)), "one for each sequence"),
    (T, "positions", Described(I, (3, 39)), "positions: expected shape"),
    (T, "mask", Described(W, (3, 40, 1)), "mask: expected shape"),
    (T, "mask", Described(W, (3, 39, 2)), "mask: expected shape"),
    (T, "slopes", Described(F, (4,)), "slopes: a contiguous one for each of the 8"),
    (T, "filter", Described(W, (4,)), "cannot hold a bit"),
    (T, "out", Described(H, (3, 40, 4, 64)), "shape of the queries"),
    (T, "lse", Described(F, (3, 8, 40)), "lse: expected shape"),
    (K, "paths", Described(I, (2, 6)), "paths: expected shape"),
    (K, "paths", Described(I, (3, 1025)), "at most 1024 entries"),
    (K, "kept", Described(I, (2,)), "one for each sequence"),
    (P, "targets", Described(I, (3,)), "one for each source"),
    (P, "keys", Described(H, (9, 17, 4, 64)), "same shape"),
    # layouts
    (A, "turns", Described(I, (5, 3), (6, 2)), "contiguous"),
    (A, "axes", Described(I, (32,), (2,)), "contiguous"),
    (D, "parents", Described(I, (3, 40), (80, 2)), "contiguous"),
    (D, "mask", Described(W, (3, 40, 2), (96, 2, 1)), "contiguous"),
    (D, "positions", Described(I, (3, 40), (48, 1)), "contiguous"),
    (D, "positions", Described(I, (3, 40), (0, 1)), "contiguous"),
    (T, "mask", Described(W, (3, 40, 2), (160, 4, 2)), "contiguous"),
    (T, "positions", Described(I, (3, 40), (80, 2)), "contiguous"),
    (T, "queries", Described(H, (3, 40, 8, 64), (20480, 512, 64, 2)), "contiguous"),
    (T, "queries", Described(H, (3, 40, 8, 64), (20480, 516, 64, 1)), "16-byte boundaries"),
    (T, "out", Described(H, (3, 40, 8, 64), (0, 512, 64, 1)), "overlap"),
    (T, "out", Described(H, (3, 40, 8, 64), (20480, 448, 64, 1)), "overlap"),
    (T, "lse", Described(F, (3, 40, 8), (400, 10, 1)), "contiguous"),
    (T, "workspace", Described(torch.uint8, (1 << 20,), address=(1 << 40) + 8), "16-byte boundary"),
    (K, "keys", Described(H, (9, 16, 4, 64), (0, 256, 64, 1)), "overlap"),
    (K, "kept", Described(I, (3,)), "lengths' own memory"),
    (K, "kept", Described(I, (3,), address=(1 << 40) + 8), "lengths' own memory"),
    (K, "kept", Described(I, (3,), address=(1 << 40) - 4), "lengths' own memory"),
    (P, "values", Described(H, (9, 16, 4, 64), (4096, 128, 64, 1)), "overlap"),
    (P, "sources", Described(I, (4,), (2,)), "contiguous"),
])
def test_refused(op, name, tensor, message):
    with pytest.raises(L.CuvsError, match=message):
        check(op, {name: tensor})


def test_what_belongs_together():
    with pytest.raises(L.CuvsError, match="turns go with frequencies"):
        check(A, {"frequencies": None})
    with pytest.raises(L.CuvsError, match="turns by 3 axes"):
        check(A, {"axes": None})
    check(A, {"axes": None, "turns": Described(I, (5, 1))})
    check(A, {"axes": None, "turns": Described(I, (5,))})
    check(A, {"turns": Described(I, (5,), (3,))})
    check(A, {"turns": Described(I, (5, 3), (0, 1))})


def test_scalars_are_checked():
    def bits(scale, cap):
        return 0, kv_cache._bits(scale), kv_cache._bits(cap)
    for scale in (float("nan"), float("inf"), -float("inf")):
        with pytest.raises(L.CuvsError, match="scale must be finite"):
            check(T, scalars=bits(scale, 0.0))
    for cap in (float("nan"), float("inf"), -1.0, 1e-38, 1e38):
        with pytest.raises(L.CuvsError, match="cap must be"):
            check(T, scalars=bits(1.0, cap))
    for cap in (1e-30, 1.0, 1e30):
        check(T, scalars=bits(-1.0, cap))
    with pytest.raises(L.CuvsError, match="window"):
        check(T, scalars=(-1, *TREE[1:]))
    check(T, scalars=(2 ** 63 - 1, *TREE[1:]))
    with pytest.raises(L.CuvsError, match="do not describe"):
        check(T, scalars=TREE[:2])
    with pytest.raises(L.CuvsError, match="unknown call"):
        L.check(L.load().cuvsB200KvCacheCheck(DEVICE, 9, *kv_cache._words([], ())))


def test_strided_shared_and_empty_tensors_pass():
    check(T, {"mask": Described(W, (3, 40, 2), (0, 2, 1)), "positions": Described(I, (3, 40), (0, 1))})       # one tree for all sequences
    check(T, {"mask": Described(W, (3, 40, 5), (0, 0, 1))})
    check(T, {"queries": Described(H, (3, 40, 8, 64), (64, 4096, 256, 1)), "out": Described(H, (3, 40, 8, 64), (64, 2048, 256, 1))})
    check(D, {"parents": Described(I, (3, 40), (0, 1))})
    check(D, {"parents": Described(I, (0, 40), address=0), "lengths": Described(I, (0,), address=0), "mask": Described(W, (0, 40, 2), address=0),
              "positions": Described(I, (0, 40), address=0)})
    check(T, {"pages": Described(I, (3, 0), address=0)})
    check(K, {"paths": Described(I, (3, 0), address=0)})
    check(K, {"paths": Described(I, (3, 6), (0, 1))})
    check(P, {"sources": Described(I, (0,), address=0), "targets": Described(I, (0,), address=0)})


def test_pages_that_are_too_large_to_be_copied():
    def page(tokens):
        t = Described(H, (2, tokens, 1, 256))
        return {"keys": t, "values": t}
    check(P, page((1 << 25) - 1))
    with pytest.raises(L.CuvsError, match="too large"):
        check(P, page(1 << 25))


def test_python_refuses_what_it_cannot_describe():
    cpu = torch.zeros((2, 16, 4, 64), dtype=H)
    ints = torch.zeros((2, 4), dtype=I)
    with pytest.raises(ValueError, match="CUDA"):
        kv_cache.draft_tree(ints, ints[:, 0])
    with pytest.raises(ValueError, match="CUDA"):
        kv_cache.keep_path(cpu, cpu, ints, ints[:, 0], ints)
    with pytest.raises(ValueError, match="CUDA"):
        kv_cache.copy_pages(cpu, cpu, ints[0], ints[0])
    with pytest.raises(ValueError, match="window"):
        kv_cache.attend_tree(cpu, cpu, cpu, None, None, None, None, window=0)
