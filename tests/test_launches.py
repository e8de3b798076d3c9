"""How the kernels are launched, by reading their sources: a launch that may begin before the kernel in front of it has ended
belongs to a kernel that waits for that one."""

import re

from flashdecode_cuda_b200.csrc.build import CSRC


def sources():
    out = {}
    for p in sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")]):
        text = re.sub(r"/\*.*?\*/", "", p.read_text(), flags=re.S)
        out[p.name] = re.sub(r"//[^\n]*", "", text)
    return out


def block(text, at):
    """The braces that open first behind ``at``, with what they hold."""
    begin = text.index("{", at)
    depth = 0
    for i in range(begin, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[begin:i + 1]
    raise AssertionError("braces do not close")


def kernels(files):
    return {m.group(1): block(text, m.end()) for text in files.values()
            for m in re.finditer(r"__global__[^;{]*?\b(\w+_kernel)\s*\(", text)}


def early_launches(files):
    """(file, kernels) of every call that may set the attribute; a kernel in a variable: all those named in the same function."""
    for name, text in files.items():
        for m in re.finditer(r"\blaunch_(?:waiting|with)\(", text):
            call = text[m.end():text.index(";", m.end())]
            if name == "common.cuh" or call.lstrip().startswith("false"):
                continue
            named = re.findall(r"\b\w+_kernel\b", call)
            if not named:
                starts = [f.start() for f in re.finditer(r"^(?:template|static|int|extern)[^;{}]*\{", text[:m.start()], flags=re.M)]
                named = re.findall(r"\b\w+_kernel\b", text[starts[-1]:m.start()])
            yield name, named


def test_kernels_that_may_begin_early_wait():
    files = sources()
    body = kernels(files)
    calls = list(early_launches(files))
    assert len(calls) > 20 and all(named for _, named in calls), calls
    for name, named in calls:
        for k in named:
            assert "pdl_wait()" in body[k], f"{name}: {k} may begin before the kernel in front of it has ended, and does not wait for it"


def test_the_plain_launch_never_begins_early():
    text = sources()["common.cuh"]
    launch = block(text, text.index("inline int launch("))
    assert "launch_with(false" in launch
    assert "g_pdl" in block(text, text.index("inline int launch_waiting("))


def test_a_launch_does_not_change_the_switch_for_others():
    """Launches of several threads at once: the switch is written where it is set, and nowhere for the length of a launch."""
    for name, text in sources().items():
        text = text.replace("extern int g_pdl", "").replace("int g_pdl = 0;", "")
        for m in re.finditer(r"\bg_pdl\s*=(?!=)", text):
            assert name == "runtime.cu" and "fd_set_pdl" in text[:m.start()][-120:], f"{name} sets g_pdl"
