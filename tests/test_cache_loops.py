"""That the rotary step's and the paged cache's kernels keep to their registers inside their loops, from the built library's code; runs without a GPU."""

import re
import shutil
import subprocess

import pytest

from ksanadit_amd import _capi

LLVM = "/opt/rocm/llvm/bin"
KERNELS = ("sage_rotary_kernel", "sage_cache_rows_kernel", "sage_cache_few_kernel", "sage_cache_join_kernel")


def in_loops(instructions: list) -> list:
    """Those of ``[(address, text)]`` that can come to themselves again: Tarjan's components of more than one instruction, or that branch to themselves."""
    number = {address: i for i, (address, _) in enumerate(instructions)}
    start = instructions[0][0]
    follow = []
    for i, (_, text) in enumerate(instructions):
        to = [] if re.match(r"s_(branch|endpgm)", text) or i + 1 == len(instructions) else [i + 1]
        if re.match(r"s_c?branch", text):
            target = re.search(r" <[^+>]+(?:\+0x([0-9a-f]+))?>$", text)
            to.append(number[start + int(target[1] or "0", 16)])
        follow.append(to)
    index, low, stacked, stack, looped, count = {}, {}, set(), [], set(), 0
    for root in range(len(follow)):
        if root in index:
            continue
        work = [(root, iter(follow[root]))]
        index[root] = low[root] = count
        count += 1
        stack.append(root)
        stacked.add(root)
        while work:
            node, rest = work[-1]
            for to in rest:
                if to not in index:
                    index[to] = low[to] = count
                    count += 1
                    stack.append(to)
                    stacked.add(to)
                    work.append((to, iter(follow[to])))
                    break
                if to in stacked:
                    low[node] = min(low[node], index[to])
            else:
                work.pop()
                if work:
                    low[work[-1][0]] = min(low[work[-1][0]], low[node])
                if low[node] == index[node]:
                    part = stack[stack.index(node):]
                    del stack[-len(part):]
                    stacked.difference_update(part)
                    if len(part) > 1 or node in follow[node]:
                        looped.update(part)
    return [instructions[i][1] for i in sorted(looped)]


def test_loops_are_found():
    code = [(0, "v_mov"), (4, "s_cbranch_scc1 2  <k+0x10>"), (8, "scratch_load_dword"), (12, "s_branch 1 <k+0x14>"), (16, "v_add"), (20, "v_mul"), (24, "s_cbranch_vccnz 3 <k+0x10>"), (28, "s_endpgm")]
    assert in_loops(code) == ["v_add", "v_mul", "s_cbranch_vccnz 3 <k+0x10>"]
    assert in_loops([(0, "v_mov"), (4, "s_branch 9 <k>")]) == ["v_mov", "s_branch 9 <k>"]


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: [(address, instruction)]}"""
    tool = shutil.which("llvm-objdump", path=LLVM)
    if tool is None or not _capi.LIB_PATH.exists():
        pytest.skip("needs the built library and ROCm's object tools")
    folder = tmp_path_factory.mktemp("objects")
    shutil.copy(_capi.LIB_PATH, folder / "lib.so")
    subprocess.run([tool, "--offloading", "lib.so"], cwd=folder, check=True, capture_output=True)
    found = {}
    for part in sorted(folder.glob("*gfx950*")):
        name = None
        for line in subprocess.run([tool, "-d", str(part)], check=True, capture_output=True, text=True).stdout.splitlines():
            head = re.match(r"[0-9a-f]+ <(\S+)>:", line)
            if head:
                name = head[1] if any(k in head[1] for k in KERNELS) else None
            elif name and (code := re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):(?: [0-9A-F]{8})+( <\S+>)?$", line)):
                found.setdefault(name, []).append((int(code[2], 16), code[1] + (code[3] or "")))
    return found


@pytest.mark.parametrize("kernel,number", [("sage_rotary_kernel", 21), ("sage_cache_rows_kernel", 8), ("sage_cache_few_kernel", 8), ("sage_cache_join_kernel", 8)])
def test_nothing_goes_through_memory_in_loops(kernels, kernel, number):
    own = {name: code for name, code in kernels.items() if kernel in name}
    assert len(own) == number
    for name, code in own.items():
        inside = in_loops(code)
        if kernel != "sage_cache_join_kernel":  # (whose loops are unrolled)
            assert sum("s_cbranch" in text for text in inside) > 0, name
        assert not [text for text in inside if text.startswith("scratch_")], name
