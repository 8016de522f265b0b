"""GPU: the LDS and resident waves registered for the kernels of expert layers and 4-bit
weights are the loaded code object's, and no kernel keeps its loop's values in scratch."""
import pytest

import pyc_amd
from pyc_amd import abi

pytestmark = pytest.mark.gpu
KEYS = ("moe_route", "moe_combine", "grouped_gemm", "matmul_w4a16", "grouped_w4a16")


def test_registered_resources_match_the_code_object(gpu):
    lib, seen = pyc_amd.lib(), 0
    for key in KEYS:
        descs = (abi.KernelDesc * 64)()
        n = lib.pyc_kernel_collect(key.encode(), abi.BACKEND_CUDA, descs, 64)
        assert n == lib.pyc_hip_kernel_symbol_count(key.encode())
        for d in descs[:n]:
            sym = d.symbol.decode()
            r = pyc_amd.kernel_resources(sym)
            assert r.device == 1, sym
            assert d.shared_mem_bytes == r.lds_bytes == r.attr_lds_bytes, (sym, r.lds_bytes, r.attr_lds_bytes)
            assert r.attr_max_threads >= r.threads, sym
            assert r.waves_per_simd == r.attr_blocks_per_cu * (r.threads // 64) / 4, (sym, r.waves_per_simd, r.attr_blocks_per_cu)
            assert abs(d.estimated_occupancy - r.waves_per_simd / 8.0) < 1e-12, sym
            assert r.attr_scratch_bytes == 0, sym
            seen += 1
    assert seen == 11
