"""CPU-only checks of rules that the 4-bit kernels' sources have to keep and no run can show."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rfx-fuse_b200", "csrc")


def _code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def _loads(text, call):
    """The arguments of every ``call(...)`` in text, parentheses balanced."""
    out = []
    for m in re.finditer(re.escape(call) + r"\(", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        out.append(text[m.end():i - 1])
    return out


def test_the_selection_reads_the_keys_in_order():
    """k_f4_pick* start while k_f4_keys may still write the keys and error bounds.  Both are read
    after the wait for it, and by ordinary loads: a non-coherent one may be moved above the wait."""
    text = _code("rfx_fp4_topk.cu")
    shared = re.compile(r"\bkeys\b|\berrs\b")
    assert not [a for a in _loads(text, "__ldg") if shared.search(a)]
    assert "ld.global.nc" not in text
    kernels = [k for k in re.split(r"__global__", text) if "wait_for_previous();" in k]
    assert len(kernels) == 2
    for k in kernels:
        before, after = k.split("wait_for_previous();")
        reads = [a for a in _loads(k, "load_left") if shared.search(a)]
        assert len(reads) >= 2 and reads == [a for a in _loads(after, "load_left") if shared.search(a)]
        # before the wait the keys' address is taken, nothing more
        assert len(re.findall(r"\bp\.errs\b", before)) == 0
        assert len(re.findall(r"\bkeys\b(?!\s*=)", before)) == len(re.findall(r"\bp\.keys\b", before)) == 1
