"""The ISA of the 8-bit training kernels, compiled as the build compiles them: no read of a load in flight, no flat access
(one counts as an access of LDS, and its waits with it), no scratch, none of the packed fp32 operations that the build turns
off. Needs hipcc, no GPU."""
import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, 'siren_amd', 'csrc')
TUS = ['tu_fp8_quant.hip', 'tu_fp8_gemm.hip', 'tu_adamw.hip']


@pytest.fixture(scope='module')
def isa(tmp_path_factory):
    hipcc = shutil.which('hipcc') or '/opt/rocm/bin/hipcc'
    if not os.path.exists(hipcc):
        pytest.skip('hipcc is not installed')
    sys.path.insert(0, ROOT)
    import __graft_entry__ as build
    tmp = tmp_path_factory.mktemp('isa')

    def compile_one(tu):
        out = str(tmp / tu.replace('.hip', '.s'))
        subprocess.check_call([hipcc, '--offload-arch=gfx950', '-O3', '-std=c++17', '-mllvm',
                               '-pragma-unroll-threshold=1000000'] + build.TU_FLAGS[tu] +
                              ['--cuda-device-only', '-S', '-I', os.path.join(ROOT, 'include'), '-o', out,
                               os.path.join(CSRC, tu)], stderr=subprocess.DEVNULL)
        return open(out).read()
    with ThreadPoolExecutor(3) as ex:
        return dict(zip(TUS, ex.map(compile_one, TUS)))


@pytest.mark.parametrize('tu', TUS)
def test_kernels_are_clean(isa, tu):
    sys.path.insert(0, os.path.join(ROOT, 'tools'))
    import check_asm_waits as C
    s, names = isa[tu], 0
    for nm in re.findall(r'\n(_Z\w+):', s):
        i = s.find('\n' + nm + ':')
        body = s[i:s.find('.Lfunc_end', i)].split('\n')
        names += 1
        for check in (C.check, C.check_vmem, C.check_store_data):
            assert not check(body, nm), (nm, check.__name__)
        assert not C.check_flat(body, nm) and not C.check_private(body, nm), nm
    assert names
    assert not re.search(r'\bv_pk_(add|mul|fma)_f32\b', s)


def test_products_use_the_matrix_pipe_and_direct_loads(isa):
    s = isa['tu_fp8_gemm.hip']
    assert 'v_mfma_f32_32x32x16_bf16' in s and 'v_cvt_scalef32_pk_bf16_fp8' in s and 'global_load_lds_dwordx4' in s
    assert 'v_cvt_scalef32_pk_fp8' in isa['tu_fp8_quant.hip']
