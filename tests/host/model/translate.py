"""Kernel sources -> C++ units that a host compiler takes: includes are laid out in order, named barriers and the waits with
inline PTX go to the models, launches become calls.  Everything else is the kernels' own text."""
import os
import re

COMMON = ['sbl_common.cuh', 'sbl_tc_host.cuh']
UNITS = {
    'gradients': ['sbl_bwd_walk.cuh', 'sbl_tc_bwd.cu'],
    'forward64': ['sbl_band_walk.cuh', 'sbl_tc.cu'],
    'forward128': ['sbl_tc128.cu'],
    'api': ['sbl_api.cu'],
}
# waits written with inline PTX in the kernels' files
BODIES = {
    'mbar_test': '  return model::mbar_test(bar, parity);',
    'wait_inline': '  model::mbar_wait(bar, parity, code);',
    'bulk_load': '  model::load_bytes(smem, src, bytes, bar);',
}


def _closing(s, i):
    """Index of the bracket that closes the one at i."""
    depth = 0
    for j in range(i, len(s)):
        depth += (s[j] == '(') - (s[j] == ')')
        if depth == 0:
            return j
    raise ValueError(s[i:i + 80])


def _arguments(s):
    out, depth, at = [], 0, 0
    for i, c in enumerate(s + ','):
        depth += (c == '(') - (c == ')')
        if c == ',' and depth == 0:
            out.append(s[at:i].strip())
            at = i + 1
    return out


def _launches(s):
    """kernel<A, B><<<grid, block, bytes, stream>>>(args) -> model::launch(grid, block, bytes, [&] { kernel<A, B>(args); })"""
    out, at = '', 0
    while (i := s.find('<<<', at)) >= 0:
        k, depth = i, 0
        while True:
            k -= 1
            depth += (s[k] == '>') - (s[k] == '<')
            if depth == 0 and s[k] in ' \n(;{':
                break
        end = s.index('>>>', i)
        close = _closing(s, end + 3)
        grid, block, size = _arguments(s[i + 3:end])[:3]
        out += s[at:k + 1] + f'model::launch({grid}, {block}, {size}, [&] {{ {s[k + 1:i]}{s[end + 3:close + 1]}; }})'
        at = close + 1
    return out + s[at:]


def translate(s):
    s = re.sub(r'^#include "[^"]*"\n', '', s, flags=re.M).replace('#pragma once', '')
    s = re.sub(r'extern __shared__ (?:__align__\(\d+\) )?(uint8_t|float) (\w+)\[\];',
               r'\1* \2 = reinterpret_cast<\1*>(model::smem);', s)
    nested = r'((?:[^()]|\([^()]*\))*)'
    s = re.sub(r'asm volatile\("bar\.sync (\d+), (\d+);" ::: "memory"\);', r'model::barrier_sync(\1, \2);', s)
    s = re.sub(r'asm volatile\("bar\.sync (\d+), %0;" ::"n"\(' + nested + r'\) : "memory"\);',
               r'model::barrier_sync(\1, \2);', s)
    s = re.sub(r'asm volatile\("bar\.sync %0, (\d+);" ::"r"\(' + nested + r'\) : "memory"\);',
               r'model::barrier_sync(\2, \1);', s)
    for name, body in BODIES.items():
        m = re.search(r'__device__ __forceinline__ \w+ ' + name + r'\([^{;]*\) \{\n', s)
        if m:
            s = s[:m.end()] + body + s[s.index('\n}\n', m.end()):]
    s = _launches(s)
    left = re.search(r'\basm\b.*', s)
    if left:
        raise ValueError(f'inline PTX that no model stands for: {left.group(0)}')
    return s


def write_units(csrc, out, change=lambda name, text: text):
    """Writes the units into `out` and returns their paths.  change: (file name, text) -> text, before the translation."""
    paths = []
    for unit, files in UNITS.items():
        text = '#include "device_model.h"\n#include "sblocal_b200.h"\n'
        for name in COMMON + files:
            with open(os.path.join(csrc, name)) as fh:
                text += translate(change(name, fh.read()))
        paths.append(os.path.join(out, unit + '.cpp'))
        with open(paths[-1], 'w') as fh:
            fh.write(text)
    return paths
