"""The kernels that stand with their entry points in .inl files are dependent launches too: each waits for the kernel ahead of it before it
reads or writes anything (the check of the .cuh files' kernels, on these)."""
import importlib
import os
import re

import pytest
from test_dependent_launches import KERNEL, _misses

SHARED_KERNELS = {"add_norm_q8_kernel": "norm_q8.inl", "adapters_kernel": "adapters.inl"}


def _body(text, at):
    start = text.index("{", at)
    depth, end = 0, start
    while True:
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        end += 1
        if depth == 0:
            return text[start:end]


def _kernels(pkg):
    bld = importlib.import_module(pkg.__name__ + ".build")
    for name in sorted(os.listdir(bld.CSRC)):
        if name.endswith(".inl"):
            text = re.sub(r"//[^\n]*", "", open(os.path.join(bld.CSRC, name)).read())
            assert len(KERNEL.findall(text)) == text.count("__global__"), name
            for m in KERNEL.finditer(text):
                yield m.group(1), name, _body(text, m.end())


def test_operator_kernels_wait_first(pkg):
    found = {k: (name, _misses(body)) for k, name, body in _kernels(pkg)}
    assert found == {k: (name, "") for k, name in SHARED_KERNELS.items()}


def test_operator_kernels_are_launched_as_dependent_ones(pkg):
    bld = importlib.import_module(pkg.__name__ + ".build")
    for name in set(SHARED_KERNELS.values()):
        text = open(os.path.join(bld.CSRC, name)).read()
        assert "launch_dependent" in text and "<<<" not in text
