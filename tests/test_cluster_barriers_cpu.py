"""Shared memory of another CTA is touched only once its cluster has met at a barrier: before that the other CTA may not have started."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alignedkv_b200", "csrc")
REMOTE = re.compile(r"(?:st|ld|red|atom)(?:\.\w+)*\.shared::cluster|mapa\b")
MET = re.compile(r"\b(?:cluster_sync|cluster_wait|sync_all)\(\)")


def bodies(text):
    """(name, body) of every function: from the brace behind its arguments to the brace that closes it."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"(\w+)\([^;{}]*\)\s*(?:const\s*)?\{", text):
        if m[1] in ("if", "for", "while", "switch"):
            continue
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        yield m[1], text[m.end():i], text[:m.start()].rfind("__global__") > max(text[:m.start()].rfind("}"), text[:m.start()].rfind(";"))


def files():
    return [f for f in sorted(os.listdir(CSRC)) if REMOTE.search(open(os.path.join(CSRC, f)).read())]


@pytest.mark.parametrize("name", files())
def test_a_barrier_comes_first(name):
    found = list(bodies(open(os.path.join(CSRC, name)).read()))
    helpers = {f for f, body, kernel in found if not kernel and REMOTE.search(body) and not MET.search(body)}      # (address or value of another CTA's variable)
    used = re.compile("|".join([REMOTE.pattern] + [rf"\b{f}\(" for f in sorted(helpers)]))
    kernels = [(f, body) for f, body, kernel in found if kernel and used.search(body)]
    assert kernels
    for f, body in kernels:
        barrier = MET.search(body)
        assert barrier and barrier.start() < used.search(body).start(), f
        # an arrival of its own is matched by its wait
        assert body.count("cluster_arrive()") == body.count("cluster_wait()"), f
