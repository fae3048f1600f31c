"""Which tiles and splits the feed-forward products choose at the sizes of the GPU tests
that are there for them (test_gpu_feed_forward_tiles.py): the estimates of the HIP sources,
compiled for the host. A change of an estimate that takes a tile out of those tests fails
here."""

import ctypes
import os
import shutil
import subprocess

import pytest

from metal_liger_amd import build

# rows, in, out of the linear layer; what its forward is: a step as the epilogue of a 256 x
# 256 tile, K split over workgroups
LINEAR_256 = (3300, 1352, 3768)
LINEAR_SPLIT = [(200, 2048, 2048), (300, 2056, 2048)]
# rows, hidden, inter, out of the gated block. The first: both projections as 256 x 256
# tiles; the second: the projection back and the gradient step so; both: the weights'
# gradients in whole rounds and tiles split over the rows; the others: all split.
MLP_256 = [(1603, 1544, 4104, 520), (3301, 264, 3768, 3768)]
MLP_SPLIT = [(200, 2048, 1024, 264), (250, 2056, 2056, 520)]
# rows, in, out in fp32 and fp16, where the forward, dX and dW are 128 x 128 tiles with K
# whole
F32_FORWARD, F32_DX, F32_DW = (1800, 264, 2056), (1800, 2056, 264), (264, 2056, 1800)

SOURCE = r"""
#include "ffn_f32.h"
#include "ffn_product.h"
#include "ffn_skinny.h"
#include "ffn_wgrad.h"
using namespace mla;
extern "C" {
int step_tile(int kind, int64_t M, int64_t columns, int64_t K) {
  return ffn::step_tile(kind, M, columns, K);
}
int splits(int64_t M, int64_t N, int64_t K) {
  const int m = (int)M, n = (int)N, kt = (int)((K + gemm::kBK - 1) / gemm::kBK);
  return gemm::plan_products(1, &m, &n, &kt, true).ksplit;
}
void f32(int64_t M, int64_t N, int64_t K, int* out) {
  const ffn::F32Plan p = ffn::plan_f32(M, N, ffn::f32_ktiles(1, &K));
  out[0] = p.tile;
  out[1] = p.splits;
}
void wgrads(int count, const int64_t* sizes, int64_t K, int* out) {
  ffn::WgradTiles t[ffn::kMaxWgrads];
  for (int i = 0; i < count; ++i) t[i] = {sizes[2 * i], sizes[2 * i + 1]};
  const ffn::WgradPlan p = ffn::plan_wgrads(count, t, K);
  out[0] = p.tiles;
  out[1] = p.full;
  out[2] = p.splits;
}
int most_rows_of_few() { return ffn::kSkinnyRows; }
int plain() { return ffn::kPlainStep; }
int act() { return ffn::kActStep; }
int pair() { return ffn::kPairStep; }
int grad() { return ffn::kGradStep; }
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    hipcc = os.environ.get("HIPCC") or shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    where = tmp_path_factory.mktemp("plans")
    (where / "plans.hip").write_text(SOURCE)
    flags = [f for f in build.HIP_FLAGS if f != "-Wall"]
    include = os.path.join(os.path.dirname(build.PKG_DIR), "include")
    subprocess.run([hipcc, *flags, "-w", "-shared", f"-I{build.CSRC_DIR}", f"-I{include}",
                    str(where / "plans.hip"), "-o", str(where / "plans.so")], check=True,
                   capture_output=True)
    return ctypes.CDLL(str(where / "plans.so"))


def _i64(*values):
    return [ctypes.c_int64(v) for v in values]


def _f32(plans, *mnk):
    out = (ctypes.c_int * 2)()
    plans.f32(*_i64(*mnk), out)
    return tuple(out)


def _wgrads(plans, K, *sizes):
    out, n = (ctypes.c_int * 3)(), len(sizes) // 2
    plans.wgrads(n, (ctypes.c_int64 * (2 * n))(*sizes), *_i64(K), out)
    return tuple(out)


def _edges(tile, *sizes):
    return all(s % tile for s in sizes)


def test_linear(plans):
    M, K, N = LINEAR_256
    assert plans.splits(*_i64(M, N, K)) == 1 and _edges(256, M, N) and K % 64
    assert plans.step_tile(plans.act(), *_i64(M, N, K)) == 256
    for M, K, N in LINEAR_SPLIT:
        assert plans.splits(*_i64(M, N, K)) > 1 and M > plans.most_rows_of_few()


def test_gated_block(plans):
    M, H, I, O = MLP_256[0]  # noqa: E741
    assert plans.splits(*_i64(M, 2 * I, H)) == 1 and _edges(256, M, I) and H % 64
    assert plans.step_tile(plans.pair(), *_i64(M, 2 * I, H)) == 256
    M, H, I, O = MLP_256[1]  # noqa: E741
    for kind in (plans.plain(), plans.grad()):  # [M, I] x O here: sizes both ways round
        assert I == O and plans.step_tile(kind, *_i64(M, I, O)) == 256
    assert plans.splits(*_i64(M, I, O)) == 1 and _edges(256, M, I)
    for M, H, I, O in MLP_256:  # noqa: E741
        tiles, full, splits = _wgrads(plans, M, I, H, I, H, O, I)
        assert 256 <= full < tiles and splits > 1 and M % 64
    for M, H, I, O in MLP_SPLIT:  # noqa: E741
        assert M > plans.most_rows_of_few()
        assert plans.splits(*_i64(M, 2 * I, H)) > 1 and plans.splits(*_i64(M, O, I)) > 1


def test_fp32(plans):
    (M, K, N), (M2, K2, N2), (M3, K3, N3) = F32_FORWARD, F32_DX, F32_DW
    for m, n, k in ((M, N, K), (M2, K2, N2), (N3, K3, M3)):
        assert _f32(plans, m, n, k) == (128, 1) and _edges(128, m, n) and k % 32
