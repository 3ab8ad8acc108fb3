"""Kernels that are launched with the programmatic attribute wait for their predecessor: read from the sources.

A kernel that follows one that signals early starts while that one still writes; only its own griddepcontrol.wait orders the
two.  So every kernel that does not go through a plain <<<>>> launch, which the stream orders by itself, has to wait, and no
thread may leave the kernel, or reach its work, around the wait."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "fastconv_b200" / "csrc"


def code(path):
    """The file without comments and string literals."""
    text = path.read_text()
    text = re.sub(r'"(\\.|[^"\\\n])*"', '""', text)
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def bodies(text, marker):
    """{function name: body} of the functions that `marker` introduces."""
    found = {}
    for m in re.finditer(marker, text):
        # the name is what stands before the first parenthesis that is not an attribute's
        rest = re.sub(r"__launch_bounds__\s*\(", lambda k: k.group().replace("(", "\x01"), text[m.end():])
        rest = re.sub(r"__cluster_dims__\s*\(", lambda k: k.group().replace("(", "\x01"), rest)
        depth, clean = 0, []
        for c in rest:  # drop the attributes' arguments
            if c == "\x01":
                depth += 1
            elif depth and c == "(":
                depth += 1
            elif depth and c == ")":
                depth -= 1
                continue
            if not depth and c != "\x01":
                clean.append(c)
            if c == "{" and not depth:
                break
        name = re.search(r"(\w+)\s*\(", "".join(clean)).group(1)
        start = rest.index("{", rest.index(name))
        level, end = 0, start
        for end in range(start, len(rest)):
            level += {"{": 1, "}": -1}.get(rest[end], 0)
            if level == 0:
                break
        found[name] = rest[start:end + 1]
    return found


def without_lambdas(body):
    """The body without named lambdas' own bodies: their returns leave the lambda."""
    while True:
        m = re.search(r"=\s*\[[&=]\]\s*\([^{};]*\)\s*\{", body)
        if not m:
            return body
        level, end = 0, m.end() - 1
        for end in range(m.end() - 1, len(body)):
            level += {"{": 1, "}": -1}.get(body[end], 0)
            if level == 0:
                break
        body = body[:m.start()] + body[end + 1:]


def kernels():
    for path in sorted(CSRC.glob("*.cu")):
        text = code(path)
        helpers = bodies(text, r"__device__(?: __forceinline__| __noinline__)*(?: static)? (?=void\b|bool\b)")
        plain = {m.group(1) for m in re.finditer(r"(\w+)\s*(?:<[^;<>]*>)?\s*<<<", text)}
        for name, body in bodies(text, r"__global__").items():
            yield path.name, name, body, helpers, name in plain


KERNELS = list(kernels())


def test_the_kernels_are_found():
    names = {k[1] for k in KERNELS}
    assert len(names) >= 40
    assert {"igemm_tiny_unfused_kernel", "norm_fused_kernel", "ff_tc_kernel", "map_move_kernel", "wino_gemm_tc_kernel", "direct_tc_kernel",
            "wino_gemm_ffma_tma_kernel", "ff_tc_join_kernel"} <= names
    for path in CSRC.glob("*.cu"):  # and none is missed
        assert code(path).count("__global__") == sum(k[0] == path.name for k in KERNELS), path.name


@pytest.mark.parametrize("file,name,body,helpers", [k[:4] for k in KERNELS if not k[4]], ids=[k[1] for k in KERNELS if not k[4]])
def test_a_kernel_of_a_programmatic_launch_waits(file, name, body, helpers):
    called = [n for n in helpers if re.search(rf"\b{n}\s*(?:<[^;{{}}]*?>)?\s*\(", body)]
    waits = [body] if "pdl_wait()" in body else [helpers[n] for n in called if "pdl_wait()" in helpers[n]]
    assert waits, f"{file}: {name} never waits for its predecessor"
    for text in waits:
        text = without_lambdas(text)
        before = text[:text.index("pdl_wait()")]
        assert not re.search(r"\breturn\s*;", before), f"{file}: threads of {name} may leave before the wait"


def test_what_an_early_kernel_may_still_write_is_not_read_through_the_read_only_path():
    """Kernels that signal early, and those that start behind them, read by plain loads; all others are launched by launch_pdl,
    which leaves the attribute out once the context has had an early kernel."""
    early = [f for f in CSRC.glob("*.cu") if "pdl_next()" in code(f)]
    assert len(early) >= 5
    for path in (*early, CSRC / "fc_last.cuh"):
        text = code(path)
        assert "__ldg" not in text and "ld.global.nc" not in text, path.name
        assert not re.search(r"const\s+\w+\s*\*\s*__restrict__", text), path.name
    assert not re.search(r"launch_pdl\s*\(", "".join(code(p) for p in early))
    moves = code(CSRC / "fc_map_move.cu")
    assert "__restrict__" not in moves  # one of the two is read, by direction
    internal, last = code(CSRC / "fc_internal.h"), code(CSRC / "fc_last.cuh")
    assert "pdl_enabled() && !ctx->signals_early" in internal and last.count("ctx->signals_early = true") == 2
    for path in CSRC.glob("*.cu"):
        if path not in early:
            assert "launch_early" not in code(path) and "launch_clusters" not in code(path) and "cudaLaunchKernelEx" not in code(path)
