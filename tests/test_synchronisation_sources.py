"""Rules of synchronisation that show in no result a test could rely on, read from the sources."""
import glob
import os
import re

from conftest import ROOT

CSRC = os.path.join(ROOT, "moe-explore_b200", "csrc")


def _sources():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        with open(path) as f:
            yield os.path.basename(path), re.sub(r"//[^\n]*", "", f.read())


def test_every_arrival_releases():
    """What a barrier guards changes hands by arrivals that release (the default): nobody is let on by one that orders nothing."""
    arrivals = [(name, a) for name, text in _sources() for a in re.findall(r"mbarrier\.arrive[\w.:]*", text)]
    assert len(arrivals) >= 4
    assert [x for x in arrivals if "relaxed" in x[1]] == []


def _closing(text, at, opening, closing):
    """The place behind the bracket that closes the one at `at`."""
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == opening) - (text[i] == closing)
        if depth == 0:
            return i + 1
    raise ValueError("brackets do not match")


def _functions():
    """(file, is a kernel, name, parameters, body) of every device function and kernel that has a body."""
    for name, text in _sources():
        for m in re.finditer(r"__(global|device)__\s", text):
            at = m.end()
            while True:
                word = re.compile(r"[^()\s]+\s*|\s+").match(text, at)
                if word is None or text[word.end():word.end() + 1] != "(" and text[word.end()] in ";={":
                    break
                at = word.end()
                if text[at] != "(":
                    continue
                end = _closing(text, at, "(", ")")
                if word.group().strip() == "__launch_bounds__":
                    at = end
                    continue
                body = re.compile(r"\s*(?:const\s*)?\{").match(text, end)
                if body:
                    stop = _closing(text, body.end() - 1, "{", "}")
                    yield name, m.group(1) == "global", word.group().strip(), text[at:end], text[body.end():stop]
                break


def test_chained_kernels_are_known_by_what_they_do():
    """Every kernel that waits for its predecessor, by whatever name the wait goes, is listed here, promises the compiler no constant
    memory and reads nothing through the read-only path: it begins while its predecessor still writes."""
    functions = list(_functions())
    waits = {name for _, kernel, name, _, body in functions if not kernel and "griddepcontrol.wait" in body}
    assert waits == {"grid_wait"}
    while True:
        more = {name for _, kernel, name, _, body in functions
                if not kernel and any(re.search(rf"\b{w}\(", body) for w in waits)} - waits
        if not more:
            break
        waits |= more
    chained = [(file, name, params, body) for file, kernel, name, params, body in functions
               if kernel and any(re.search(rf"\b{w}\(", body) for w in waits)]
    assert {(file, name) for file, name, _, _ in chained} == {
        ("gemm_kernel.cuh", "grouped_gemm_kernel"), ("gemm_t_kernel.cuh", "grouped_gemm_kernel"), ("rows.cu", "copy_rows_kernel"),
        ("rows.cu", "dispatch_rows_kernel"), ("rows.cu", "combine_topk_kernel"), ("rows.cu", "combine_bwd_tokens_kernel"),
        ("router.cu", "router_backward_kernel"), ("f8_gemm.cu", "f8_rows_kernel"), ("f8_gemm.cu", "f8_gather_kernel"),
        ("f8_gemm.cuh", "f8_wide_kernel"), ("f8_gemm.cuh", "f8_lanes_kernel")}
    for _, _, params, body in chained:
        assert "__restrict__" not in params and "__ldg" not in body
