"""What the tcgen05 prompt kernel may do under the tail of the kernel before it and with tables that do not fit (read from its source: a race or a write behind a
buffer does not show itself in every run)."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "questwend_b200", "csrc")


def kernel(file, name):
    """(parameters, body) of a kernel."""
    with open(os.path.join(CSRC, file)) as f:
        text = f.read()
    at = re.search(r"__global__[^;{]*?\b" + name + r"\(", text).end()
    end, depth = at, 1
    while depth:
        depth += {"(": 1, ")": -1}.get(text[end], 0)
        end += 1
    parameters, begin, depth = text[at:end - 1], text.index("{", end), 0
    for i in range(begin, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return parameters, text[begin + 1:i]


def block_so_far(text, at):
    """What stands before this place in the innermost block around it."""
    depth = 0
    for i in range(at - 1, -1, -1):
        depth += {"}": 1, "{": -1}.get(text[i], 0)
        if depth < 0:
            return text[i + 1:at]
    return text[:at]


def test_the_prompt_kernel_reads_the_table_that_the_kernel_before_it_writes_at_l2():
    """``kv4_read`` writes the page table while the prompt kernel's blocks are already there: not through the read-only path."""
    parameters, body = kernel("attention_tc.cu", "attn_tc_prefill_kernel")
    declared, = [p for p in parameters.split(",") if p.split()[-1] == "page_table"]
    assert "__restrict__" not in declared
    reads = re.findall(r"(\w*\(?)pages(?: \+|\[)", body)
    assert reads and all(r == "__ldcg(" for r in reads)


def test_a_block_of_the_prompt_kernel_that_has_nothing_to_do_waits_all_the_same():
    """In a step that brings nothing all blocks are such: the grid must not end before the kernel that it was launched under."""
    _, body = kernel("attention_tc.cu", "attn_tc_prefill_kernel")
    before = body[:body.index("pdl_launch_dependents()")]
    returns = [m.start() for m in re.finditer(r"\breturn;", before)]
    assert len(returns) >= 3 and all("pdl_wait();" in block_so_far(before, at) for at in returns)


def test_the_prompt_kernel_writes_no_row_behind_the_tokens_that_there_are():
    for name in ("attn_tc_prefill_kernel", "attn_tc_join_kernel"):
        _, body = kernel("attention_tc.cu", name)
        assert re.search(r"n_new = min\(cu_seqlens\[b \+ 1\], (T|rows / heads)\) - t0", body), name
