"""Kernels launched behind one another (csrc/launch.cuh), by their source: each waits for the kernel
before it as its first statement, and promises the compiler nothing about memory that a kernel of the
same call writes. __restrict__ on such a pointer would allow loads through it to move above the wait
or to take the path for data that never changes."""
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, 'colabfold-legacy-kernels_b200', 'csrc')
# the caller's own inputs, which no kernel of a call writes
INPUTS = {'ids', 'dout', 'labels', 'x'}


def source(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r'//[^\n]*', '', text)


def kernels(text):
    """{name: (parameters, body)} of the __global__ functions."""
    found = {}
    for m in re.finditer(r'__global__[^;{]*?(\w+_kernel)\s*\(', text):
        at, depth = m.end(), 1
        while depth:
            depth += {'(': 1, ')': -1}.get(text[at], 0)
            at += 1
        params, start = text[m.end():at - 1], text.index('{', at) + 1
        end, depth = start, 1
        while depth:
            depth += {'{': 1, '}': -1}.get(text[end], 0)
            end += 1
        found[m.group(1)] = (params, text[start:end])
    return found


FILES = sorted(f for f in os.listdir(CSRC)
               if f.endswith('.cu') and 'launch.cuh' in source(f))


def chained(text):
    """The kernels that wait for one before them."""
    return {k: v for k, v in kernels(text).items() if 'wait_before()' in v[1]}


def test_files_are_found():
    assert {'embed.cu', 'linear_xent.cu', 'xent_few.cu', 'xent_head.cu'} <= set(FILES)


@pytest.mark.parametrize('name', FILES)
def test_a_kernel_launched_behind_another_waits_first(name):
    text = source(name)
    launched = set(re.findall(r'launch_behind\(\s*(\w+_kernel)', text))
    if re.search(r'launch_behind\(\s*kern\b', text):
        launched |= set(re.findall(r'auto kern = (\w+_kernel)', text))
    assert launched
    for k in launched:
        assert re.match(r'\s*wait_before\(\);', kernels(text)[k][1]), k


@pytest.mark.parametrize('name', FILES)
def test_no_promise_about_memory_that_the_chain_writes(name):
    for k, (params, _) in chained(source(name)).items():
        for p in params.split(','):
            if '__restrict__' in p:
                assert p.split()[-1] in INPUTS and 'const' in p, '%s: %s' % (k, p.strip())
