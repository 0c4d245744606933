"""What inline assembly has to guarantee by itself, from listings of small kernels compiled for gfx950 (no GPU needed)."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'tensorgrad_amd', 'csrc')
HIPCC = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')

# A base that a vector instruction puts into scalar registers, and loads from there straight into LDS at once.
SOURCE = '''
#include "attend_dev.h"
using namespace tgk;
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t x = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return (const char*)((uint64_t)hi << 32 | lo);
}
__global__ void fragments(const char* const* at, float* y) {
  __shared__ __align__(16) float lds[8192];
  frags_to_lds<8>(uniform(at[threadIdx.x]), lds_address(lds), 16 * threadIdx.x, 0);
  loads_done();
  y[threadIdx.x] = lds[threadIdx.x];
}
template <bool DW>
__global__ void tiles(const char* const* at, float* y) {
  using T = gd::DTile<64, 32, true, 256, DW>;
  __shared__ __align__(16) float lds[T::SIZE];
  uint32_t off[T::PER];
  T::offsets(32, 1, 0, 64, threadIdx.x, off);
  T::dma((const float*)uniform(at[threadIdx.x]), off, lds_address(lds), 0);
  loads_done();
  y[threadIdx.x] = lds[threadIdx.x];
}
template __global__ void tiles<false>(const char* const*, float*);
template __global__ void tiles<true>(const char* const*, float*);
'''
# wait states between a vector instruction that writes a scalar register and what reads it
LOAD, VECTOR = 5, 2


def scalars(operand):
    m = re.fullmatch(r's\[(\d+):(\d+)\]|s(\d+)|(m0)', operand)
    if not m:
        return set()
    if m[4]:
        return {'m0'}
    return set(range(int(m[1]), int(m[2]) + 1)) if m[1] else {int(m[3])}


def short_waits(listing):
    """(instructions of inline assembly that are looked at, those whose scalar operands a vector instruction wrote too short before)."""
    looked, short, before, inside = 0, [], [], False   # before: what each instruction's vector result is, and its wait states
    for line in listing.splitlines():
        inside = (inside or '#ASMSTART' in line) and '#ASMEND' not in line
        words = line.split(';')[0].replace(',', ' ').split()
        if not words or words[0].startswith('.') or words[0].endswith(':'):
            continue
        op, states, wrote = words[0], 1, set()
        load = op.startswith('global_load_lds')
        if load or (inside and op.startswith('v_')):
            looked += 1
            reads, waited = ({'m0'} if load else set()).union(*map(scalars, words[1 if load else 2:])), 0
            for w, n in reversed(before):
                if w & reads:
                    short.append((waited, line.strip()))
                    break
                waited += n
                if waited >= (LOAD if load else VECTOR):
                    break
        if op == 's_nop':
            states = int(words[1], 0) + 1
        elif op.startswith('v_'):
            wrote = scalars(words[1]) | (scalars(words[2]) if '_co_' in op or op.startswith(('v_mad_u64', 'v_mad_i64', 'v_div_scale')) else set())
        before.append((wrote, states))
    return looked, short


def listing_of(source, out):
    subprocess.run([HIPCC, '--offload-arch=gfx950', '-O3', '-std=c++17', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops', '-w',
                    '--cuda-device-only', '-S', '-I', CSRC, str(source), '-o', str(out)], check=True)
    return out.read_text()


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason='no compiler')
def test_loads_into_lds_wait_for_scalars_that_vector_instructions_wrote(tmp_path):
    """The compiler does not look into assembly: a load that reads such a register too early takes its old value."""
    src = tmp_path / 'k.hip'
    src.write_text(SOURCE)
    loads, short = short_waits(listing_of(src, tmp_path / 'k.s'))
    assert loads >= 1 + 2 + 8 and not short, short


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason='no compiler')
def test_products_with_scalar_coefficients_wait_for_them(tmp_path):
    """k_sample.hip's series takes its coefficients from scalar registers, in assembly."""
    products, short = short_waits(listing_of(os.path.join(CSRC, 'k_sample.hip'), tmp_path / 'k.s'))
    assert products > 100 and not short, short[:4]


def test_the_count_of_wait_states():
    early = 'v_readlane_b32 s13, v90, 9\ns_nop 0\nglobal_load_lds_dwordx4 v2, s[12:13]\n'
    assert short_waits(early) == (1, [(1, 'global_load_lds_dwordx4 v2, s[12:13]')])
    assert short_waits(early.replace('s_nop 0', 's_nop 4')) == (1, [])
    assert short_waits(early.replace('s13', 's14')) == (1, [])
    assert short_waits('v_readfirstlane_b32 m0, v1\ns_nop 3\nglobal_load_lds_dword v[2:3], off\n')[1] == [(4, 'global_load_lds_dword v[2:3], off')]
    series = '\t;;#ASMSTART\nv_fma_f64 v[0:1], v[0:1], v[2:3], s[4:5]\n\t;;#ASMEND\n'
    assert short_waits('v_readlane_b32 s4, v9, 0\n' + series)[1] and not short_waits('v_readlane_b32 s4, v9, 0\ns_nop 1\n' + series)[1]
