"""Dependent launches and loads, in the sources: a kernel that starts while the kernel
before it may still write its inputs must not read them as read-only memory.

`ld.global.nc` and `__ldg` say that the memory is read-only as long as the kernel runs,
and for `const T* __restrict__` parameters the compiler may use the same loads, and move
them above the wait.
"""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "inference-kernel_b200" / "csrc"


def code(path: Path) -> str:
    """The source without comments."""
    text = re.sub(r"/\*.*?\*/", "", path.read_text(), flags=re.S)
    return re.sub(r"//[^\n]*", "", text)


def functions_with(text: str, call: str):
    """(signature, body) of the top-level functions whose body holds `call`."""
    found = []
    for m in re.finditer(r"__global__", text):
        brace = text.index("{", m.start())
        if ";" in text[m.start():brace]:
            continue
        depth, end = 0, brace
        for end in range(brace, len(text)):
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            if depth == 0:
                break
        body = text[brace:end]
        if call in body:
            found.append((text[m.start():brace], body))
    return found


SOURCES = sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")])
DEPENDENT = [p for p in SOURCES if p.suffix == ".cu" and "pdl_wait_prior()" in code(p)]


def test_the_dependent_kernels_are_found():
    names = {p.name for p in DEPENDENT}
    assert {"mxfp4.cu", "sandwich_norm.cu", "rmsnorm.cu", "activation.cu", "gemm_tc.cu", "gemm_tc2.cu",
            "gemm_skinny.cu", "gemm_mxfp4.cu", "gemm_mxfp4_skinny.cu"} <= names
    for p in DEPENDENT:
        assert functions_with(code(p), "pdl_wait_prior()"), p.name


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_no_read_only_loads(path):
    text = code(path)
    assert not re.search(r"ld\.global[\w.:]*\.nc\b", text) and "__ldg(" not in text
    assert "ld.global.nc" not in text


@pytest.mark.parametrize("path", DEPENDENT, ids=lambda p: p.name)
def test_inputs_of_dependent_kernels_are_not_restrict(path):
    for signature, _ in functions_with(code(path), "pdl_wait_prior()"):
        for param in signature.split(","):
            assert not ("const" in param and "*" in param and "__restrict__" in param), param


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_loads_in_statements_are_volatile(path):
    """One that is not volatile may be executed ahead of the condition that guards it."""
    for m in re.finditer(r"\basm\s*(volatile)?\s*\(", code(path)):
        text = code(path)[m.end():]
        text = text[:text.index(";\n")]
        if re.search(r'"[^"]*\bld\.', text):
            assert m.group(1), text
