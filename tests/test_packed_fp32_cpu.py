"""The kernel libraries hold no packed fp32 arithmetic: hipcc makes it from scalar code by itself, and some of its forms have given wrong
results on this hardware."""
import os
import re
import struct
import subprocess

import pytest
import torch

from gast_hip import binding

LLVM = os.path.join(os.environ.get('ROCM_PATH', '/opt/rocm'), 'llvm', 'bin')
MAGIC = b'__CLANG_OFFLOAD_BUNDLE__'


def device_code(library, tmp):
    """the gfx950 code objects of a library, one for each source"""
    section = str(tmp / 'fatbin')
    subprocess.run([os.path.join(LLVM, 'llvm-objcopy'), '--dump-section', '.hip_fatbin=' + section, library, os.devnull], check=True)
    with open(section, 'rb') as f:
        data = f.read()
    for m in re.finditer(MAGIC, data):
        at = m.end()
        count, = struct.unpack_from('<Q', data, at)
        at += 8
        for _ in range(count):
            offset, size, n = struct.unpack_from('<QQQ', data, at)
            triple = data[at + 24:at + 24 + n].decode()
            at += 24 + n
            if 'gfx950' in triple:
                yield data[m.start() + offset:m.start() + offset + size]


@pytest.mark.skipif(not os.path.exists(os.path.join(LLVM, 'llvm-objdump')), reason='no llvm-objdump')
@pytest.mark.parametrize('h16', [torch.bfloat16, torch.float16], ids=['bf16', 'f16'])
def test_no_packed_fp32_instructions(h16, tmp_path):
    objects = 0
    for i, code in enumerate(device_code(binding.library_path(h16), tmp_path)):
        path = tmp_path / ('%d.co' % i)
        path.write_bytes(code)
        text = subprocess.run([os.path.join(LLVM, 'llvm-objdump'), '-d', str(path)], check=True, capture_output=True, text=True).stdout
        assert 's_endpgm' in text
        found = re.findall(r'\bv_pk_(?:add|mul|fma)_f32\b', text)
        assert not found, '%d in source %d' % (len(found), i)
        objects += 1
    assert objects >= 13


def test_the_load_hazard_screens_hold_for_the_flags_of_the_build(tmp_path):
    """scripts/asm_load_hazard.py on the sources with loads in inline asm, compiled as csrc/build.sh compiles them (gemm_big and wgrad_wide, which
    take minutes, with GAST_TEST_ASM_SCAN_ALL=1)"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    csrc = os.path.join(root, 'gast-net-3dposeestimation_amd', 'csrc')
    hipcc = '/opt/rocm/bin/hipcc'
    if not os.path.exists(hipcc):
        pytest.skip('no hipcc')
    with open(os.path.join(csrc, 'build.sh')) as f:
        flags = re.search(r'^FLAGS="([^"$]*)"', f.read(), re.M).group(1).split()
    assert '-packed-fp32-ops' in flags
    names = ['gemm', 'wgrad', 'gemm_bj'] + (['gemm_big', 'wgrad_wide'] if os.environ.get('GAST_TEST_ASM_SCAN_ALL') else [])
    runs = []
    for n in names:
        out = str(tmp_path / (n + '.s'))
        runs.append((n, out, subprocess.Popen([hipcc] + flags + ['-S', '--cuda-device-only', os.path.join(csrc, n + '.hip'), '-o', out], stdout=subprocess.DEVNULL,
                                              stderr=subprocess.PIPE)))
    for n, out, p in runs:
        _, err = p.communicate(timeout=900)
        assert p.returncode == 0, '%s.hip did not compile: %s' % (n, err.decode()[-800:])
        for mode, none in (('--strict', '0 suspicious instruction(s)'), ('--sgpr', '0 VALU->SGPR->VMEM hazard(s)')):
            r = subprocess.run(['python3', os.path.join(root, 'scripts', 'asm_load_hazard.py'), mode, out], capture_output=True, text=True)
            assert r.returncode == 0 and none in r.stdout, '%s.hip: %s' % (n, r.stdout[-1500:])
