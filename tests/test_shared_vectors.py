"""CPU test of the kernels' source: no element of a vector in LDS is assigned by itself. The compiler may load the whole vector, insert the
element and store the whole, which between waves that write one element each loses the others' (an array of floats has no such reading)."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stream-_amd", "csrc")


def element_writes(text):
    """names of __shared__ arrays of vectors that text assigns to with one subscript more than they are declared with"""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)
    vectors = set(re.findall(r"using\s+(\w+)\s*=\s*[\w ]+__attribute__\(\(ext_vector_type", text)) | {"f4", "u2", "u4", "f16v", "s4"}
    bad = []
    for attrs, kind, names in re.findall(r"__shared__\s+((?:__attribute__\(\(.*?\)\)\s*)?)(\w+)\s+([^;]*);", text):
        if kind not in vectors:
            continue
        for name, subscripts in re.findall(r"(\w+)((?:\[[^\]]*\])+)", names):
            more = subscripts.count("[") + 1
            if re.search(r"\b%s(?:\[[^\]]*\]){%d}\s*(?:[-+*/|&^]|<<|>>)?=[^=]" % (name, more), text):
                bad.append(name)
    return bad


def test_the_search():
    declared = "__shared__ f4 a[2], b; __shared__ __attribute__((aligned(16))) float c[2][4];"
    assert element_writes(declared + "a[i][w] = 1;") == ["a"]
    assert element_writes(declared + "a[i] = x; c[i][w] = 1; y = a[i][w] == 2;") == []


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.h*"))), ids=os.path.basename)
def test_no_element_of_a_shared_vector_is_written(path):
    with open(path) as f:
        assert element_writes(f.read()) == []
