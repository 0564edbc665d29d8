"""What the layer kernels' sources have to keep to, read as text: rules whose
breach could hang the GPU or race, which no run would show for sure."""
import os
import re

CUDA = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc", "cuda")


def code(name):
    """The source without comments."""
    with open(os.path.join(CUDA, name)) as f:
        text = f.read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def kernel(text, name):
    """The body of a __global__ function."""
    start = text.index("{", text.index(name + "("))
    depth = 0
    for i in range(start, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[start:i + 1]
    raise AssertionError("no end")


def test_a_warp_gives_up_as_one():
    """A wait that runs out is a decision of the whole warp: a warp of which some
    lanes leave and some go on to the warp-wide loads of tensor memory hangs."""
    body = kernel(code("dense_gemm.cuh"), "k_gemm")
    statements = [" ".join(s.split()) for s in re.split(r"[;{}]", body)]
    waits = [s for s in statements if "wait_bar" in s and "kDrainNs" not in s]
    assert len(waits) >= 4
    for s in waits:
        assert re.search(r"__all_sync\(kFull, .*wait_bar", s), s
    for s in statements:
        if re.search(r"\*aborted\b(?! = 1)", s) and "const aborted" not in s:
            assert "__all_sync(kFull" in s, s


def test_no_copy_outlives_its_cta():
    """However the loads' warp ends (all copies issued, or a wait given up, its own
    or another warp's), it leaves only when its copies have landed: it waits for
    the products that read the last of them, else for a fixed time."""
    body = kernel(code("dense_gemm.cuh"), "k_gemm")
    loads = body[body.index("if (warp == 0)"):body.index("else if (warp == 1")]
    tail = " ".join(loads[loads.index("++loads"):].split())
    issued = tail.index("wait_bar(empty(")  # behind the loop, over the last kStages loads
    gave_up = tail.index("if (!ok)")
    assert issued < gave_up and "loads - S::kStages" in tail[:issued] and "ok = __all_sync" in tail[:issued]
    assert re.search(r"globaltimer\(\) - t0 < kDrainNs", tail[gave_up:])
    assert "rank" not in tail  # both CTAs of a pair


def test_dependent_launches_read_with_ordinary_loads():
    """A programmatic dependent lives while the kernel in front still writes, so
    nothing may come over the read-only path (its memory must not change while
    the kernel lives), and no load may move in front of the wait: ordinary loads
    behind its memory clobber, or volatile asm with one of its own."""
    names = [n for n in os.listdir(CUDA) if n.startswith(("dense", "norm", "layer"))]
    assert len(names) > 10
    for n in names:
        text = code(n)
        assert "__ldg" not in text and "__restrict__" not in text, n
        for m in re.finditer(r"asm\s*(volatile)?\s*\(", text):
            end = text.index(";\n", m.end())
            statement = text[m.start():end]
            assert ".nc" not in statement, (n, statement)
            if re.search(r"\bld\.global|griddepcontrol", statement):
                assert m.group(1) and '"memory"' in statement, (n, statement)
