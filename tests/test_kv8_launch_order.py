"""Kernels of the paged 8-bit cache are launched while the one before them still runs.  What that one and its
predecessors wrote is promised to them behind their wait alone, so every one of them waits first, whatever the batch."""
import pathlib
import re

import pytest

KERNELS = pathlib.Path(__file__).resolve().parent.parent / "bladedisc_b200" / "csrc" / "kernels"


def kernels(name):
    """(name, body without comments) of every __global__ function of a source file."""
    text = re.sub(r"//[^\n]*", "", (KERNELS / name).read_text())
    for m in re.finditer(r"__global__\s+void\b", text):
        kernel = re.search(r"(\w+)\s*\((?!\w*,\s*\d\))", text[m.end():].replace("__launch_bounds__", "")).group(1)
        at = text.index("{", m.end())
        depth, end = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield kernel, text[at + 1:end - 1]


def statements(body):
    """Statements of a function's outermost level, those of inner blocks as part of them."""
    depth, at = 0, 0
    for i, c in enumerate(body):
        depth += {"{": 1, "(": 1, "}": -1, ")": -1}.get(c, 0)
        if depth == 0 and c in ";}":
            yield body[at:i + 1].strip()
            at = i + 1


def first_wait(body):
    """The outermost statements before the first unconditional wait, or None if there is none."""
    before = []
    for s in statements(body):
        if s == "grid_dep_wait();":
            return before
        before.append(s)
    return None


@pytest.mark.parametrize("name", ["kv_blocks.cu", "kv8_cache.cu", "kv8_attention.cu", "kv8_prefill.cu"])
def test_every_kernel_waits_before_it_goes_on(name):
    found = list(kernels(name))
    assert found
    for kernel, body in found:
        before = first_wait(body)
        assert before is not None, f"{kernel} reads without waiting for the kernel before it"
        text = "\n".join(s for s in before if not s.startswith("auto "))  # lambdas return to the kernel
        assert "return" not in text and "grid_dep" not in text and "_body" not in text, kernel
        assert body.count("grid_dep_wait") == 1, f"{kernel} waits in two places"


def test_the_reading_of_sources_finds_a_missing_wait():
    assert first_wait("int a = f(1); grid_dep_wait(); g();") == ["int a = f(1);"]
    assert first_wait("if (x) fence();\n else grid_dep_wait(); g();") is None
    assert first_wait("if (x) { grid_dep_wait(); }") is None
