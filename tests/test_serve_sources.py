"""Rules of the serving sources that one GPU cannot show."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tcb_b200", "csrc")
FILES = ["tcb_serve.cu", "tcb_page_decode.cu", "tcb_page_rows.cu", "tcb_logits.cu", "tcb_page.h"]


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", FILES)
def test_function_attributes_are_asked_for_on_every_device(name):
    """An attribute belongs to the kernel on one device: a result kept in a
    static would leave every other device without it."""
    statements = re.split(r"[;{}]", source(name))
    kept = [s for s in statements if re.search(r"\bstatic\b.*\bcuda(FuncSetAttribute|Error_t)\b", s, re.S)]
    assert not kept, kept


def kernels():
    for name in FILES:
        for body in re.split(r"__global__", source(name))[1:]:
            if "{" in body:
                yield name, re.search(r"\b(k_\w+)\(", body).group(1), body


@pytest.mark.parametrize("name,kernel,body", [pytest.param(*k, id=k[1]) for k in kernels()])
def test_kernels_wait_before_they_touch_memory(name, kernel, body):
    """The launches allow a kernel to start before the last one has ended, and
    what earlier kernels wrote is promised to threads that have waited alone: every
    kernel waits, whatever its arguments, before its first access."""
    body = body[body.index("{"):]
    at = body.index("pdl_wait()")
    line = body[body.rindex("\n", 0, at) + 1:body.index("\n", at)]
    assert line.strip() in ("mv::pdl_wait();", "tcb::mv::pdl_wait();") and len(line) - len(line.lstrip()) == 2, line
    before = body[:at]
    for access in (r"\ba\.\w+\s*\[", r"[(=,]\s*\*\s*a\.", r"atomic\w+\(", r"__ld\w+\(", r"reinterpret_cast<const uint4", r"tma_load\(", r"\btables?\["):
        assert not re.search(access, before), access
