"""GPU tests of which kernel takes the 8-bit products of few rows: the streaming one, whose
work-groups walk all of K, up to 10240 columns of K (6144 above 16 rows), k ranges of tiles beyond."""
import pytest
import torch

from my_pytchon_opencl_lib_amd import _native
from test_int8_gpu import check, int8, product64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k,plan", [
    (8, 64, 131056, "int8-tiles"), (1, 16, 65536, "int8-tiles"), (16, 500, 16384, "int8-tiles"),
    (8, 300, 10256, "int8-tiles"), (8, 300, 10240, "int8-rows"), (24, 64, 8192, "int8-tiles"),
    (32, 70, 6160, "int8-tiles"), (32, 70, 6144, "int8-rows"), (16, 2048, 8208, "int8-rows"),
    (24, 2048, 6016, "int8-rows"), (1, 17, 48, "int8-rows")])
def test_long_k_of_few_columns_is_cut(nncl, m, n, k, plan):
    print(m, n, k, flush=True)
    a, b = int8(m + k, m, k), int8(n + k + 1, n, k)
    sa, sb = torch.rand(m, device="cuda") + 0.1, torch.rand(n, device="cuda") + 0.1
    got = nncl.MatmulInt8(a, sa, b, sb)
    assert _native.last_plan().startswith(plan + " "), _native.last_plan()
    check(got, *product64(a, sa, b, sb))
