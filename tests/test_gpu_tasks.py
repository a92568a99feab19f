"""The numbering of the prompt attention's tiles (``sgld_attend.cuh``), in any order of the numbers: a
kernel compiled here asks for them one after another, as a block that claims waiting blocks does."""
import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(shutil.which("nvcc") is None, reason="nvcc not available")]
ROOT = Path(__file__).resolve().parents[1]
SOURCE = r"""
#include "sgld_attend.cuh"
using namespace sgld;
// One warp: tiles[0 .. n) in that order with one cursor; per tile valid, q0, q1, k0, k1, index.
__global__ void find(const __grid_constant__ AttendLaunch a, int step, const int* tiles, int n, int* found) {
  int chunk = 0;
  int64_t before = 0;
  for (int i = 0; i < n; ++i) {
    int r[6] = {0, 0, 0, 0, 0, 0};
    r[0] = find_tile(a, step, tiles[i], chunk, before, r[1], r[2], r[3], r[4], r[5]) ? 1 : 0;
    if (threadIdx.x == 0)
      for (int x = 0; x < 6; ++x) found[i * 6 + x] = r[x];
  }
}
extern "C" int run(const int* q_indptr, const int* kv_indptr, int tokens, int keys, int seqs, int window, int step,
                   const int* tiles, int n, int* found) {
  AttendLaunch a = {};
  a.q_indptr = q_indptr, a.kv_indptr = kv_indptr;
  a.tokens = tokens, a.kv_count = keys, a.seqs = seqs, a.window_left = window;
  find<<<1, 32>>>(a, step, tiles, n, found);
  return static_cast<int>(cudaDeviceSynchronize());
}
"""


@pytest.fixture(scope="module")
def find(tmp_path_factory):
    folder = tmp_path_factory.mktemp("tasks")
    (folder / "tasks.cu").write_text(SOURCE)
    subprocess.run(["nvcc", "-gencode=arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "-shared", "-Xcompiler", "-fPIC",
                    "-diag-suppress=177", f"-I{ROOT / '-sglang-decode-_b200' / 'csrc'}", f"-I{ROOT / 'include'}",
                    str(folder / "tasks.cu"), "-o", str(folder / "tasks.so")], check=True)
    lib = ctypes.CDLL(str(folder / "tasks.so"))
    lib.run.argtypes = [ctypes.c_void_p] * 2 + [ctypes.c_int] * 5 + [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    return lib.run


def pointers(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).int().cuda()


@pytest.mark.parametrize("order", ["ascending", "descending", "shuffled"])
@pytest.mark.parametrize("seqs", [1, 2, 33, 128, 129, 150, 700])
def test_every_tile_is_found_once_in_any_order(cuda_device, find, seqs, order):
    rng = random.Random(seqs)
    step, window = 64, -1
    q_lens = [rng.choice([0, 1, 2, 63, 64, 65, 200, 500]) for _ in range(seqs)]
    kv_lens = [n + rng.choice([0, 3, 200, -40]) for n in q_lens]
    kv_lens = [max(n, 0) for n in kv_lens]
    want = set()
    q0 = k0 = 0
    for n, m in zip(q_lens, kv_lens):
        want |= {(q0, q0 + n, k0, k0 + m, i) for i in range(-(-n // step))}
        q0, k0 = q0 + n, k0 + m
    numbers = list(range(len(want) + 5))          # those past the last are none
    if order == "descending":
        numbers.reverse()
    if order == "shuffled":
        rng.shuffle(numbers)
    tiles = torch.tensor(numbers, dtype=torch.int32, device="cuda")
    found = torch.zeros(len(numbers), 6, dtype=torch.int32, device="cuda")
    q_indptr, kv_indptr = pointers(q_lens), pointers(kv_lens)
    assert find(q_indptr.data_ptr(), kv_indptr.data_ptr(), max(q0, 1), max(k0, 1), seqs, window, step, tiles.data_ptr(),
                len(numbers), found.data_ptr()) == 0
    rows = [tuple(r) for r in found.tolist()]
    assert [bool(r[0]) for r in rows] == [n < len(want) for n in numbers]
    got = [r[1:] for r in rows if r[0]]
    assert len(got) == len(want) and set(got) == want
