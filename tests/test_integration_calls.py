"""The calls that the integration document shows, against the declarations of tsr_hip.h: as many arguments, and those that carry a
parameter's name in its place. No GPU calls."""
import os
import re

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def arguments(text, at):
    """The arguments of the call whose parenthesis opens at text[at], split at its own commas."""
    depth, args, cur = 0, [], ""
    for ch in text[at:]:
        if ch in "([{":
            depth += 1
            if depth == 1:
                continue
        elif ch in ")]}":
            depth -= 1
            if depth == 0:
                return [a.strip() for a in args + [cur] if a.strip()]
        if ch == "," and depth == 1:
            args, cur = args + [cur], ""
        else:
            cur += ch
    return None


def test_calls_fit_their_declarations():
    with open(os.path.join(REPO, "include", "tsr_hip.h")) as f:
        header = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    params = {}
    for m in re.finditer(r"\b(tsr_hip_\w+)\(", header):
        args = arguments(header, m.end() - 1)
        params[m[1]] = [re.sub(r"\W", " ", re.sub(r"\[\d+\]", "", a)).split()[-1] for a in args]
    with open(os.path.join(REPO, "INTEGRATION.md")) as f:
        doc = f.read()
    seen = 0
    for m in re.finditer(r"\b(tsr_hip_\w+)\(ctx,", doc):
        args = arguments(doc, m.end() - 5)
        assert m[1] in params, m[1]
        want = params[m[1]]
        assert len(args) == len(want), (m[1], args, want)
        for i, a in enumerate(args):
            if a in want:
                assert want.index(a) == i, (m[1], a, want)
        seen += 1
    assert seen > 20
