"""Shared arrays of fixed size that kernels read or write by vectors are declared for it: an array of 4-byte elements is on a boundary of 4 by its type, and
whether the compiler happens to place it on 16 is seen in no test's results until it does not."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "seq2seqsharp_b200", "csrc")
BYTES = {"float4": 16, "uint4": 16, "int4": 16, "double2": 16, "longlong2": 16, "ulonglong2": 16, "float2": 8, "uint2": 8, "int2": 8, "double": 8, "uint64_t": 8, "int64_t": 8}
SIZES = {"float": 4, "int": 4, "unsigned": 4, "uint32_t": 4, "__half": 2, "unsigned char": 1, "uint8_t": 1, "uint16_t": 2, "double": 8, "float2": 8, "float4": 16, "uint4": 16, "uint64_t": 8}


def misdeclared(text):
    text = re.sub(r"//[^\n]*", "", text)
    found = []
    for d in re.finditer(r"(extern\s+)?__shared__\s+(__align__\((\d+)\)\s+)?(unsigned char|\w+)\s+([^;]*\[[^;]*);", text):
        if d.group(1):
            continue                                          # the size of the launch: such memory begins on a boundary of 16
        size = max(int(d.group(3) or 0), SIZES.get(d.group(4), 16))
        for name in re.findall(r"(\w+)\s*(?:\[[^\[\]]*\]\s*)+(?:,|$)", re.sub(r"\(uintptr_t\)", "", d.group(5))):
            for c in re.finditer(r"reinterpret_cast<\s*(?:const\s+)?(\w+)\s*\*>\(\s*&?%s\b" % re.escape(name), text):
                if BYTES.get(c.group(1), 1) > size:
                    found.append((name, c.group(1)))
    return found


@pytest.mark.parametrize("file", sorted(os.path.basename(f) for f in glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))))
def test_shared_arrays_are_aligned_for_their_vectors(file):
    with open(os.path.join(CSRC, file)) as fh:
        assert misdeclared(fh.read()) == []


def test_the_check_itself():
    use = "*reinterpret_cast<float4*>(acc[share][at]) = x;"
    assert misdeclared("__shared__ float acc[W > 1 ? W : 1][4];" + use) == [("acc", "float4")]
    assert misdeclared("__shared__ __align__(16) float acc[W > 1 ? W : 1][4];" + use) == []
    assert misdeclared("__shared__ float other[4], acc[8];" + use) == [("acc", "float4")]
    assert misdeclared("__shared__ float4 acc[8];" + use) == []
