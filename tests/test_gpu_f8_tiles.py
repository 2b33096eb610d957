"""gemmF8's form for many tokens with more tiles than pairs of SMs, so that a pair computes several: results staged and stored while the next
tile's products are under way, scales handed on from tile to tile, weights' scales reloaded after 32 blocks."""
import pytest

from .test_gpu_f8 import run_gemm

pytestmark = pytest.mark.gpu


# 160 tiles of 256 x 256 and more, for 74 pairs; 1, 2, 3, 5, 33 and 37 blocks of k
@pytest.mark.parametrize("M,N,K,epi,bias,ld", [
    (2600, 3904, 100, "f16", False, 0), (2600, 3900, 128, "f32", True, 0), (2555, 4088, 256, "f16", True, 0), (2555, 4092, 300, "f32", False, 4096),
    (2600, 3896, 520, "f16", False, 3912), (2600, 3900, 640, "f32", True, 0), (2305, 4104, 4200, "f16", True, 0), (2305, 4096, 4700, "f32", False, 0),
    # rows that end or start inside of 16 bytes
    (2600, 3901, 640, "f16", False, 0), (2600, 3901, 520, "f32", True, 0), (2600, 3900, 300, "f16", False, 3901), (2305, 3842, 4200, "f16", True, 0)])
def test_plain(g, M, N, K, epi, bias, ld):
    run_gemm(g, M, N, K, epi, bias=bias, ylay=dict(ld=ld, off=0))


# 165 tiles of 256 x 128 and more
@pytest.mark.parametrize("M,N,K,epi", [(2600, 1920, 100, "geglu"), (2600, 1900, 300, "swiglu"), (2570, 1925, 640, "geglu"), (2305, 2100, 4700, "swiglu")])
def test_gated(g, M, N, K, epi):
    run_gemm(g, M, N, K, epi)


# rows of k that end inside of the first 16 bytes: one block, most of it beyond the matrix
@pytest.mark.parametrize("K", [1, 5, 17])
@pytest.mark.parametrize("M,epi", [(20, "f16"), (20, "geglu"), (100, "f32"), (1100, "f16"), (1100, "swiglu")])
def test_short_rows(g, M, K, epi):
    run_gemm(g, M, 1300, K, epi)
