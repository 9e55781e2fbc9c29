"""The chunked prefill of the linear attention (csrc/lin_prefill.cu): what comes before what in a block, as a graph.  The rows behind a sequence's end may be another
one's and hold NaN; warps clear them in k and v, and no product may read either before that.  Which barriers the clearing warps arrive at behind the
clearing, and which ones each product's warp waits for before it issues the product, is the source's; the rest of the edges is the model's.  No GPU."""
import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(__file__), "..", "glm53f-afd_b200", "csrc", "lin_prefill.cu")


def between(text, start, end):
    return text.split(start, 1)[1].split(end, 1)[0]


def waits(text):
    return re.findall(r"wait\((b[A-Z]\w*)", text)


def source():
    """Barriers arrived at behind the clearing; barriers waited for before P V of a chunk, and before w V K."""
    with open(SOURCE) as f:
        text = f.read()
    clearing = between(text, "auto weigh_values", "if (idle) goto done;").split("make_uint4(0u, 0u, 0u, 0u);", 1)[1]
    score = between(text, "} else if (warp == kScoreMmaWarp) {", "} else if (warp == kDecayWarp) {")
    # The products with V come a chunk behind the scores, in a branch of their own.
    behind = score.rsplit("if (c > 0) {", 1)[1].split("mma_bf16_if", 1)[0]
    state = between(text, "} else if (warp == kStateMmaWarp) {", "} else if (warp == kScoreMmaWarp) {")
    add = state.rsplit("mma_tf32_ts_if", 1)[1].split("mma_bf16_ts_if", 1)[0]
    return re.findall(r"arrive\((b[A-Z]\w*)", clearing), ["bP", *waits(behind)], waits(add)


def edges(chunks, after_clearing, before_pv, before_add):
    """(before, after): ("barrier", c) is its completion for chunk c."""
    out = []
    for c in range(chunks):
        out += [(("full", c), ("scores", c)), (("bP", c - 1), ("scores", c)), (("scores", c), ("bQK", c)), (("bQK", c), ("P", c)), (("P", c), ("bP", c))]
        out += [(("full", c), ("q", c)), (("bQS", c - 1), ("q", c)), (("bOFree", c - 2), ("q", c)), (("q", c), ("bReady", c)), (("add", c - 1), ("bReady", c))]
        out += [(("bReady", c), ("SQ", c)), (("SQ", c), ("bQS", c)), (("bQS", c), ("scaled", c)), (("scaled", c), ("bAdd", c)), (("bU", c - 2), ("clear", c)), (("full", c), ("clear", c))]
        out += [(("add", c), ("bU", c)), (("PV", c), ("bO", c)), (("bO", c), ("out", c)), (("out", c), ("bOFree", c))]
        out += [(("clear", c), (b, c)) for b in after_clearing] + [((b, c), ("PV", c)) for b in before_pv] + [((b, c), ("add", c)) for b in before_add]
    return out


def ordered(pairs, first, then):
    follow = {}
    for a, b in pairs:
        follow.setdefault(a, []).append(b)
    seen, todo = set(), [first]
    while todo:
        at = todo.pop()
        if at == then:
            return True
        if at not in seen:
            seen.add(at)
            todo += follow.get(at, [])
    return False


def acyclic(pairs):
    before = {}
    for a, b in pairs:
        before.setdefault(b, set()).add(a)
        before.setdefault(a, set())
    while before:
        free = [x for x, deps in before.items() if not deps & before.keys()]
        if not free:
            return False
        for x in free:
            del before[x]
    return True


def test_the_model_finds_a_product_that_does_not_wait():
    assert not ordered(edges(4, ["bAdd"], ["bP", "bQS"], ["bAdd"]), ("clear", 3), ("PV", 3))
    assert ordered(edges(4, ["bAdd"], ["bP", "bQS"], ["bAdd"]), ("clear", 3), ("add", 3))


@pytest.mark.parametrize("chunks", [1, 2, 3, 4, 7])
def test_foreign_rows_are_cleared_before_a_product_reads_them(chunks):
    pairs, last = edges(chunks, *source()), chunks - 1
    assert acyclic(pairs)  # nothing waits for what comes behind it
    assert ordered(pairs, ("clear", last), ("PV", last))
    assert ordered(pairs, ("clear", last), ("add", last))
