"""The units of the clipped step and of the 4-bit matrices, as the compiler reports them."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'deepipr_amd', 'csrc')


@pytest.mark.parametrize('unit', ['deepipr_gradnorm.hip', 'deepipr_mx4.hip'])
def test_no_kernel_spills_and_no_packed_fp32(unit, tmp_path):
    """The 256 x 256 product holds 256 accumulators and two sets of fragments a lane: a spill would be silent, right and slow."""
    out = subprocess.run(['/opt/rocm/bin/hipcc', '--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-ffp-contract=off', '-Xclang',
                          '-target-feature', '-Xclang', '-packed-fp32-ops', '--cuda-device-only',
                          '-Rpass-analysis=kernel-resource-usage', '-S', '-o', str(tmp_path / 'k.s'), os.path.join(CSRC, unit)],
                         capture_output=True, text=True, cwd=str(tmp_path))
    assert out.returncode == 0, out.stderr[-2000:]
    names = re.findall(r'Function Name: (\S+)', out.stderr)
    scratch = [int(v) for v in re.findall(r'ScratchSize \[bytes/lane\]: (\d+)', out.stderr)]
    assert len(names) == len(scratch) >= 10
    assert not {n: s for n, s in zip(names, scratch) if s}
    assert not re.findall(r'v_pk_(?:add|mul|fma)_f32', open(tmp_path / 'k.s').read())
