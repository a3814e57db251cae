"""CPU tests of attention over a paged cache: what the entry points refuse (their checks alone, no GPU), and where positions lie,
bad pages included (the kernels' own function, compiled for the host)."""
import os
import subprocess

import pytest
import torch

from cuvs_b200 import _lib as L
from cuvs_b200 import kv_cache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEVICE = 3


class Described:
    """A device tensor that is only described: type, shape, strides and an address."""

    def __init__(self, dtype, shape, strides=None, address=1 << 40, device=DEVICE):
        self.dtype, self.shape, self._address, self._device = dtype, tuple(shape), address, device
        dense = [1] * len(shape)
        for i in range(len(shape) - 2, -1, -1):
            dense[i] = dense[i + 1] * shape[i + 1]
        self._strides = tuple(strides or dense)

    def dim(self):
        return len(self.shape)

    def get_device(self):
        return self._device

    def data_ptr(self):
        return self._address

    def stride(self):
        return self._strides


H = torch.float16


def described(op):
    """The tensors of a good call, by name, and its scalars."""
    cache = {"keys": Described(H, (9, 16, 4, 64)), "values": Described(H, (9, 16, 4, 64))}
    if op == kv_cache._APPEND:
        return {**cache, "new_keys": Described(H, (5, 4, 64)), "new_values": Described(H, (5, 4, 64)),
                "pages": Described(torch.int32, (3, 7)), "positions": Described(torch.int32, (5,)),
                "sequences": Described(torch.int32, (5,)), "queries": Described(H, (5, 8, 64)),
                "frequencies": Described(torch.float64, (32,)), "slots": Described(torch.int64, (5,)),
                "rotated": Described(H, (5, 8, 64))}, (0,)
    if op == kv_cache._ATTENTION:
        return {**cache, "queries": Described(H, (3, 8, 64)), "pages": Described(torch.int32, (3, 7)),
                "lengths": Described(torch.int32, (3,)), "filter": Described(torch.uint32, (5,)), "out": Described(H, (3, 8, 64)),
                "lse": Described(torch.float32, (3, 8)), "workspace": Described(torch.uint8, (1 << 20,))}, (0, kv_cache._bits(0.125))
    if op == kv_cache._CANDIDATES:
        return {**cache, "queries": Described(H, (3, 8, 64)), "candidates": Described(torch.int64, (3, 8, 20)),
                "filter": Described(torch.uint32, (5,)), "out": Described(H, (3, 8, 64)),
                "lse": Described(torch.float32, (3, 8))}, (kv_cache._bits(0.125),)
    return {"parts": Described(H, (2, 3, 8, 64)), "parts_lse": Described(torch.float32, (2, 3, 8)), "out": Described(H, (3, 8, 64)),
            "lse": Described(torch.float32, (3, 8))}, ()


def check(op, changes=None, scalars=None):
    tensors, usual = described(op)
    tensors.update(changes or {})
    words = kv_cache._words(tensors.values(), usual if scalars is None else scalars)
    L.check(L.load().cuvsB200KvCacheCheck(DEVICE, op, *words))


OPS = [kv_cache._APPEND, kv_cache._ATTENTION, kv_cache._CANDIDATES, kv_cache._MERGE]
A, T, N, M = OPS


@pytest.mark.parametrize("op", OPS)
def test_good_calls_pass_and_calls_without_a_tensor_do_not(op):
    check(op)
    optional = {"filter", "workspace"} | ({"sequences", "frequencies"} if op == A else set())
    for name in described(op)[0]:
        if name in optional:
            if name != "sequences":
                check(op, {name: None})
        else:
            with pytest.raises(L.CuvsError, match="null tensor|together"):
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
    (A, "new_keys", Described(torch.bfloat16, (5, 4, 64)), "element type"),
    (T, "queries", Described(torch.float32, (3, 8, 64)), "element type"),
    (T, "keys", Described(torch.float64, (9, 16, 4, 64)), "unsupported element type"),
    (T, "lengths", Described(torch.int64, (3,)), "expected int32"),
    (T, "pages", Described(torch.int64, (3, 7)), "expected int32"),
    (T, "filter", Described(torch.int32, (5,)), "expected uint32"),
    (T, "lse", Described(H, (3, 8)), "expected float32"),
    (N, "candidates", Described(torch.int32, (3, 8, 20)), "expected int64"),
    (A, "slots", Described(torch.int32, (5,)), "expected int64"),
    (A, "frequencies", Described(torch.int32, (32,)), "float64 or float32"),
    # shapes that do not go together
    (A, "values", Described(H, (9, 16, 4, 56)), "same shape"),
    (A, "new_values", Described(H, (4, 4, 64)), "expected 5 rows"),
    (A, "new_keys", Described(H, (5, 3, 64)), "of 4 heads"),
    (A, "positions", Described(torch.int32, (4,)), "one for each token"),
    (A, "rotated", Described(H, (5, 4, 64)), "expected 5 rows of 8"),
    (A, "frequencies", Described(torch.float64, (33,)), "33 pairs do not fit"),
    (A, "sequences", None, "one token for each of the 3 sequences"),
    (A, "rotated", None, "together"),
    (T, "queries", Described(H, (3, 6, 64)), "no multiple"),
    (T, "queries", Described(H, (3, 0, 64)), "no multiple"),
    (T, "queries", Described(H, (3, 8, 72)), "rows of 64 elements"),
    (T, "pages", Described(torch.int32, (2, 7)), "a row for each"),
    (T, "out", Described(H, (2, 8, 64)), "out: expected 3 rows"),
    (T, "lse", Described(torch.float32, (8, 3)), "lse: expected shape"),
    (T, "filter", Described(torch.uint32, (4,)), "cannot hold a bit"),
    (T, "keys", Described(H, (9, 0, 4, 64)), "same shape"),
    (N, "candidates", Described(torch.int64, (3, 4, 20)), "a list for each"),
    (M, "parts_lse", Described(torch.float32, (2, 8, 3)), "one for each row"),
    (M, "out", Described(H, (3, 8, 56)), "shape of one part"),
    # layouts
    (T, "keys", Described(H, (9, 16, 4, 64), (4096, 256, 64, 2)), "contiguous"),
    (T, "keys", Described(H, (9, 16, 4, 64), (4104, 256, 68, 1)), "16-byte boundaries"),
    (T, "keys", Described(H, (9, 16, 4, 64), address=(1 << 40) + 8), "16-byte boundaries"),
    (T, "lse", Described(torch.float32, (3, 8), (1, 3)), "contiguous"),
    (T, "out", Described(H, (3, 8, 64), (0, 64, 1)), "overlap"),
    (A, "keys", Described(H, (9, 16, 4, 64), (0, 256, 64, 1)), "overlap"),
    (A, "values", Described(H, (9, 16, 4, 64), (4096, 128, 64, 1)), "overlap"),
    (N, "candidates", Described(torch.int64, (3, 8, 20), (320, 40, 2)), "contiguous"),
    (T, "workspace", Described(torch.uint8, (1 << 20,), address=(1 << 40) + 8), "16-byte boundary"),
    (T, "lengths", Described(torch.int32, (3,), address=(1 << 40) + 2), "boundary of its elements"),
    (A, "frequencies", Described(torch.float64, (32,), address=(1 << 40) + 4), "boundary of its elements"),
    (N, "candidates", Described(torch.int64, (3, 8, 20), address=(1 << 40) + 4), "boundary of its elements"),
    # rows at odd multiples of 16 bytes, farther than 2^32 of them reach; at multiples of 2 KB they may
    (T, "keys", Described(H, (1 << 20, 16, 4, 8), (1 << 20, 8, 128, 1)), "same shape"),
])
def test_refused(op, name, tensor, message):
    with pytest.raises(L.CuvsError, match=message):
        check(op, {name: tensor})


def test_long_and_ragged_rows_are_refused():
    for dim, message in ((264, "1 to 256"), (68, "16-byte"), (4, "16-byte")):
        with pytest.raises(L.CuvsError, match=message):
            check(M, {"parts": Described(H, (2, 3, 8, dim)), "out": Described(H, (3, 8, dim))})


def test_caches_that_places_of_32_bits_cannot_reach_are_refused():
    def with_pages(n, page):
        t = Described(H, (n, 16, 4, 64), (page, 64, 1024, 1))
        return {"keys": t, "values": t, "filter": None}
    check(T, with_pages(1 << 20, 4096))                                     # 8 GB
    check(T, with_pages(1 << 24, 8192))                                     # 256 GB, rows at multiples of 128 bytes
    with pytest.raises(L.CuvsError, match="too large for rows at multiples of 16 bytes"):
        check(T, with_pages(1 << 24, 8192 + 8))
    with pytest.raises(L.CuvsError, match="too large for rows at multiples of 128 bytes"):
        check(T, with_pages((1 << 31) - 1, 8192))


def test_scalars_are_checked():
    for scale in (float("nan"), float("inf"), -float("inf")):
        with pytest.raises(L.CuvsError, match="finite"):
            check(T, scalars=(0, kv_cache._bits(scale)))
        with pytest.raises(L.CuvsError, match="finite"):
            check(N, scalars=(kv_cache._bits(scale),))
    with pytest.raises(L.CuvsError, match="window"):
        check(T, scalars=(-1, kv_cache._bits(1.0)))
    with pytest.raises(L.CuvsError, match="do not describe"):
        check(T, scalars=(0,))


def test_strided_and_empty_tensors_pass():
    # heads of a page apart, both halves of one allocation, a table that is part of a wider one, parts of a fused projection
    check(T, {"keys": Described(H, (9, 16, 4, 64), (8192, 64, 1024, 1)), "values": Described(H, (9, 16, 4, 64), (8192, 64, 1024, 1)),
              "pages": Described(torch.int32, (3, 7), (50, 1)), "queries": Described(H, (3, 8, 64), (1024, 64, 1))})
    check(T, {"keys": Described(H, (0, 16, 4, 64), address=0), "values": Described(H, (0, 16, 4, 64), address=0),
              "filter": Described(torch.uint32, (0,), address=0)})
    check(T, {"pages": Described(torch.int32, (3, 0), address=0)})
    check(N, {"candidates": Described(torch.int64, (3, 8, 0), address=0)})
    check(N, {"candidates": Described(torch.int64, (3, 8, 0), (8, 1, 1), address=0)})
    check(M, {"parts": Described(H, (0, 3, 8, 64), address=0), "parts_lse": Described(torch.float32, (0, 3, 8), address=0)})
    check(T, {"queries": Described(H, (1, 8, 64), (7, 64, 1)), "pages": Described(torch.int32, (1, 7)), "lengths":
              Described(torch.int32, (1,)), "out": Described(H, (1, 8, 64)), "lse": Described(torch.float32, (1, 8))})


def test_python_refuses_what_it_cannot_describe():
    cpu = torch.zeros((2, 16, 4, 64), dtype=H)
    with pytest.raises(ValueError, match="CUDA"):
        kv_cache.attention(cpu, cpu, cpu[0], torch.zeros((16, 1), dtype=torch.int32), torch.zeros(16, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        kv_cache.merge_parts(cpu, cpu[..., 0].float())
    with pytest.raises(TypeError, match="expected torch tensors, not ndarray"):
        kv_cache._call(None, 0, M, (cpu.numpy(), None), 0, 0.0, False)
    with pytest.raises(ValueError, match="window"):
        kv_cache.attention(cpu, cpu, cpu[0], None, None, window=0)
    with pytest.raises(ValueError, match="element type"):
        kv_cache._words([torch.zeros(3, dtype=torch.bool)], ())
    with pytest.raises(ValueError, match="dimensions"):
        kv_cache._words([torch.zeros((1, 1, 1, 1, 1))], ())


PLACES = r"""
#include "kv_place.hpp"
#include <cassert>
#include <cstdio>
#include <vector>
using namespace cuvs_b200::kv;
int main()
{
  // pages that are none (negative, behind the last), the last page, entries behind the table's end
  const int32_t row[] = {5, -1, 0, 8, 9, 2147483647, -2147483647 - 1, 3};
  for (uint32_t size : {1u, 3u, 16u, 20u, 64u}) {
    const page_divisor by = divisor_of(size);
    for (int64_t at = -3; at < int64_t(size) * 10; at++) {
      const int64_t column = at < 0 ? 0 : at / size;
      const bool there     = at >= 0 && column < 8 && row[column] >= 0 && row[column] < 9;
      assert(slot_of(row, 8, int32_t(at), by, 9) == (there ? row[column] * int64_t(size) + at % size : -1));
      assert(slot_of(row, 0, int32_t(at), by, 9) == -1);
      assert(slot_of(row, 8, int32_t(at), by, 0) == -1);
    }
  }
  assert(slot_of(row, 8, 2147483647, divisor_of(1u << 28), 9) == 3ll * (1 << 28) + (1 << 28) - 1);   // slots behind 2^29
  const int32_t far[] = {2147483646};
  assert(slot_of(far, 1, 63, divisor_of(64), 2147483647) == 2147483646ll * 64 + 63);                   // slots behind 2^32
  // the product that stands for the division: around multiples of the size, up to the last position
  for (uint32_t size : {1u, 2u, 3u, 5u, 7u, 20u, 24u, 100u, 641u, 65535u, 65536u, 65537u, 1000003u, (1u << 30) - 1, 1u << 30, (1u << 30) + 1, 2147483647u}) {
    const page_divisor by = divisor_of(size);
    for (uint64_t k = 0; k * size < (uint64_t(1) << 31) + size; k += 1 + (uint64_t(1) << 31) / size / 4096) {
      for (int64_t at = int64_t(k * size) - 1; at <= int64_t(k * size) + 1; at++) {
        if (at < 0 || at >= int64_t(1) << 31) { continue; }
        uint32_t page, place;
        split_place(uint32_t(at), by, page, place);
        assert(page == uint32_t(at) / size && place == uint32_t(at) % size);
      }
    }
    uint32_t page, place;
    split_place(2147483647u, by, page, place);
    assert(page == 2147483647u / size && place == 2147483647u % size);
  }
  uint32_t first, end;
  attended(-5, 0, 4, 16, first, end);  assert(first == 0 && end == 0);
  attended(0, 7, 4, 16, first, end);   assert(first == 0 && end == 0);
  attended(50, 0, 4, 16, first, end);  assert(first == 0 && end == 50);
  attended(50, 50, 4, 16, first, end); assert(first == 0 && end == 50);
  attended(50, 49, 4, 16, first, end); assert(first == 1 && end == 50);
  attended(50, 1, 4, 16, first, end);  assert(first == 49 && end == 50);
  attended(99, 0, 4, 16, first, end);  assert(first == 0 && end == 64);                       // no further than the table
  attended(99, 40, 4, 16, first, end); assert(first == 59 && end == 64);
  attended(99, 10, 4, 16, first, end); assert(first == end);                                   // all of the window behind it
  attended(99, int64_t(1) << 60, 4, 16, first, end); assert(first == 0 && end == 64);
  attended(2147483647, 0, 2147483647, 2147483647, first, end); assert(end == 2147483647u);
  std::puts("ok");
}
"""


def test_places_of_positions_and_bad_pages(tmp_path):
    src, exe = tmp_path / "places.cpp", tmp_path / "places"
    src.write_text(PLACES)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "cuvs_b200", "csrc"), "-I",
                    "/usr/local/cuda/include", str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout == "ok\n"
