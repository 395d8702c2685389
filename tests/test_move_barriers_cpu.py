"""Every thread of a block meets a block-wide barrier at the same place of the source: the moving kernel's turn between reading and
writing is taken in no branch that some of its warps alone take."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "leankv_b200", "csrc")


def _functions(text):
    """Name -> body of the functions at the namespace's level."""
    out, at = {}, 0
    for m in re.finditer(r"\b(\w+)\([^;{}]*\)\s*\{", text):
        if m.start() < at:
            continue
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        name = m.group(1)
        if name == "__launch_bounds__":
            name = re.search(r"(\w+)\(const", m.group(0)).group(1)
        out[name], at = text[m.end(): i - 1], i
    return out


def _branches(body, at):
    """The conditions in force at a place of a function's body: of the blocks around it, and of its own statement."""
    heads, start = [], 0
    for i, c in enumerate(body[:at]):
        if c == "{":
            heads.append(body[start:i].strip())
        elif c == "}":
            heads.pop()
        if c in ";{}":
            start = i + 1
    own = body[start:at]
    return [h for h in heads if not h.startswith("if constexpr") and h != "else"] + re.findall(r"\b(?:if|else|for|while)\b|\?|&&|\|\|", own)


def test_no_barrier_under_a_branch():
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "tq_move.cu")).read())
    functions = _functions(text)
    kernel = functions["move_kernel"]
    waits = {"__syncthreads", "__syncthreads_or"}
    for _ in functions:
        waits |= {n for n, body in functions.items() if any(re.search(rf"\b{w}\b", body) for w in waits)}
    assert {"move_turn", "move_block_q8"} <= waits
    # an `else` without its `if constexpr` would be a branch at run time: there is none in the kernel around blocks
    assert all(re.search(r"if constexpr[^{]*\{", kernel[: m.start()]) for m in re.finditer(r"\}\s*else\s*\{", kernel))
    found = 0
    for name in waits - {"__syncthreads", "__syncthreads_or", "move_kernel", "launch_move", "run"}:
        for m in re.finditer(rf"\b{name}\b(?:<[^>;]*>)?\(", kernel):
            found += 1
            assert not _branches(kernel, m.start()), (name, _branches(kernel, m.start()))
    assert found >= 2
    # in the turn itself the branch before its last barrier is the whole block's: there are flags, or none
    assert functions["move_turn"].count("__syncthreads") == 2
