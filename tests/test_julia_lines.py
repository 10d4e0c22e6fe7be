"""Julia ends an expression at the end of a line where it is complete, and reads
the next line as another one: a line outside all brackets that begins with a
binary operator does not parse (or, with + or -, is an expression of its own).
Julia is not installed here, so the sources of julia/src are checked for that
line by line, and for brackets that do not close."""
import os
import re

import pytest

from test_julia_binding import JL

SRC = os.path.join(JL, "src")
FILES = sorted(f for f in os.listdir(SRC) if f.endswith(".jl"))
# what a statement cannot begin with (it can with :x, !x, ~x, <:T, ::T, @m)
OPERATOR = re.compile(r"(=|[*/÷%^&|⊗⨷∘+>?,)\]}-]|<(?!:)|\.[*/+^=-])")


def blank(text):
    """text with strings, character literals and comments as blanks; lines are kept."""
    tokens = r"""#=.*?=#|\"\"\".*?\"\"\"|"(?:[^"\\\n]|\\.)*"|(?<![\w)\]}])'(?:[^'\\\n]|\\.)+'|#[^\n]*"""
    return re.sub(tokens, lambda m: re.sub(r"[^\n]", " ", m.group(0)), text, flags=re.S)


def faults(text):
    """The numbers of the lines that begin with an operator outside all brackets, and
    the depth of brackets at the end."""
    depth, bad = 0, []
    for n, line in enumerate(blank(text).splitlines(), 1):
        s = line.strip()
        if depth == 0 and OPERATOR.match(s):
            bad.append(n)
        for ch in s:
            depth += (ch in "([{") - (ch in ")]}")
    return bad, depth


@pytest.mark.parametrize("name", FILES)
def test_no_line_begins_with_an_operator(name):
    assert faults(open(os.path.join(SRC, name)).read()) == ([], 0)


def test_such_lines_are_seen():
    assert faults("f(a,\n  b)\n=\n  g(a)\n") == ([3], 0)
    assert faults("f(a)\n    = g(a)\n") == ([2], 0)
    assert faults("x = a\n* b\n") == ([2], 0)
    assert faults("f(a, # )\n  '(' == \")\"\n") == ([], 1)
    assert faults("f(a,\n  b) =\n  g(a,\n    *)\n\"\"\"\n= a docstring\n\"\"\"\n# = a comment\nx'\n") == ([], 0)
