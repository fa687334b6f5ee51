"""CPU test of an order the sources must keep: a kernel that allocates TMEM lets
its dependents start only behind the allocation and a barrier of its CTA.

tcgen05.alloc waits until the columns are free. A dependent kernel that fits
beside a CTA of the kernel, and that allocates before it waits for it, could
take all columns first: the CTA then waits for the dependent and the dependent
for the CTA."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onnx_runtime_dart_b200", "csrc")


def _kernels():
    """(file:line, text) of every __global__ function that allocates TMEM."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        starts = [m.start() for m in re.finditer(r"^__global__|(?<=\n)template <[^>]*>\n__global__", text, re.M)]
        for a, b in zip(starts, starts[1:] + [len(text)]):
            body = text[a:b]
            if re.search(r"\btmem_alloc\(", body):
                yield f"{os.path.basename(path)}:{text.count(chr(10), 0, a) + 1}", body


KERNELS = list(_kernels())


def test_kernels_are_found():
    assert {k.split(":")[0] for k, _ in KERNELS} >= {"k_glue.cu", "k_kv8_flash.cu", "k_nbits_ts.cu", "k_f32_tc.cu"}


@pytest.mark.parametrize("body", [b for _, b in KERNELS], ids=[k for k, _ in KERNELS])
def test_dependents_start_behind_the_allocation(body):
    alloc = body.index("tmem_alloc(")
    for m in re.finditer(r"pdl_launch_dependents\(\)", body):
        assert m.start() > alloc and "__syncthreads()" in body[alloc: m.start()]
