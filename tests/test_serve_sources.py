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
