"""A wait on a barrier asks for the parity of one phase, so whoever waits must not fall two phases behind.  The walk over shared prefixes (csrc/attention_prefix.cu) keeps
its two chains within one phase of one another by turns: no chain says that its turn is over without having waited for it.  Read from the source, so that it needs no GPU."""
import re

from test_launch_waits import kernels


def turns(body: str):
    """For every arrival at ``exp_done``: whether a turn was waited for in the same block of statements, or in one around it that does not lie outside the loop's half."""
    taken, out = [False], []
    for m in re.finditer(r"[{}]|if\s*\(\s*!\s*take_turn\s*\(\s*j\s*,\s*n\s*\)\s*\)|mbar_arrive\s*\(\s*&\s*exp_done", body):
        token = m.group(0)
        if token == "{":
            taken.append(False)
        elif token == "}":
            taken.pop()
        elif token.startswith("if"):
            taken[-1] = True
        else:
            out.append(taken[-1])
    return out


def test_the_reader_itself():
    assert turns("{ if (a) { if (!take_turn(j, n)) { break; } mbar_arrive(&exp_done[u]); } else { mbar_arrive(&exp_done[u]); } }") == [True, False]


def test_no_turn_ends_that_was_not_waited_for():
    body = next(body for _, name, body in kernels() if name == "prefix_walk_kernel")
    assert turns(body) == [True, True]
    assert re.search(r"auto take_turn = .*?mbar_wait\(&exp_done\[u \^ 1\], turn & 1, abort_p\)", body, re.S)
