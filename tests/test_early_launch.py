"""CPU check, by reading the sources, of the kernels that are launched with programmatic stream
serialisation (csrc/kv4_attention.cuh, `launch_early`).

Such a kernel is ordered behind the one before it by its own griddepcontrol.wait alone, and what follows it in
the stream is ordered behind it alone.  So each of its CTAs has to wait, in every call: before it reads what
an earlier kernel wrote, and before it returns, or the grid could complete while the one before it
still stores its results.
"""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "long-context-attention-kernels_b200" / "csrc"
SOURCES = ["kv4_cache.cu", "kv4_attention.cu", "kv4_chunk.cu"]


def kernels(text):
    """(name, body) of every __global__ function."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"__global__", text):
        open_at = text.index("{", m.end())
        name = re.findall(r"(\w+)\s*\(const \w+ p", text[m.end():open_at])[-1]
        depth, at = 1, open_at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield name, text[open_at + 1:at - 1]


def faults(body):
    """What comes before the first unconditional wait of a kernel."""
    depth, wait = 0, None
    for m in re.finditer(r"[{}]|ptx::griddep_wait\(\);", body):
        if m.group() == "{":
            depth += 1
        elif m.group() == "}":
            depth -= 1
        elif depth == 0:
            wait = m.start()
            break
    if wait is None:
        return ["no wait that every CTA reaches"]
    before = body[:wait]
    found = ["a return before the wait"] if re.search(r"\breturn\b", before) else []
    # arrays of the call's parameters, by index or through the functions that read the lengths
    if re.search(r"\bp\.\w+\s*\[|\b(request_of|share_of|locate|item_of)\b", before):
        found.append("memory read before the wait")
    return found


def all_kernels():
    return [pytest.param(name, body, id=name) for f in SOURCES for name, body in kernels((CSRC / f).read_text())]


def test_every_kernel_is_found():
    names = [p.id for p in all_kernels()]
    assert sorted(names) == sorted(["kv_layout", "kv_release", "kv4_append", "kv4_read", "kv4_attention",
                                    "kv4_attention_merge", "kv4_chunk"])


@pytest.mark.parametrize("name,body", all_kernels())
def test_every_cta_waits_before_it_reads_or_returns(name, body):
    assert faults(body) == []


def test_the_check_notices():
    good = "int i = p.batch; ptx::griddep_wait(); if (!p.cuts[i]) return;"
    assert faults(good) == []
    assert faults("if (x) { ptx::griddep_wait(); } return;")
    assert faults("if (x) return; ptx::griddep_wait();")
    assert faults("int n = p.cu[0]; ptx::griddep_wait();")
    assert faults("const Request r = request_of(p, 0); ptx::griddep_wait();")
