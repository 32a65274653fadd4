"""Kernels whose bounded waits are reported through the library's error word, from their sources: the word's address is null where the driver did not give it, and nothing may be written there then."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "seq2seqsharp_b200", "csrc")


def sources():
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            text = f.read()
        if re.search(r"=\s*tc_error_word\(", text) and name != "gemm_tc.cu":
            yield name, text


@pytest.mark.parametrize("name,text", list(sources()), ids=[name for name, _ in sources()])
def test_error_word_is_looked_at_before_it_is_written(name, text):
    writes = re.findall(r"^.*\*\s*((?:\w+\.)?(?:error|error_flag))\s*=[^=].*$", text, re.M)
    lines = [line for line in text.splitlines() if re.search(r"\*\s*(?:\w+\.)?(?:error|error_flag)\s*=[^=]", line)]
    assert len(writes) == len(lines)
    for word, line in zip(writes, lines):
        condition = re.search(r"if \((.*)\)\s*\*", line)
        assert condition and re.search(r"(?<![\w.])" + re.escape(word) + r"(?!\w)", condition.group(1)), "%s: %s" % (name, line.strip())
