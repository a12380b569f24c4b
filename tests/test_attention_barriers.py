"""The order that barriers give the 16-bit gradients' keys walk, from its source: a stage of shared memory is written anew only when every
row warp has read what lies in it."""
import re
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parent.parent / "torchpairwise_b200" / "csrc" / "attention_backward.cu"


def keys_walk():
    text = SOURCE.read_text()
    return text[text.index("void keys_walk("):text.index("void queries_walk(")]


def section(text, first, last):
    start = text.index(first)
    return text[start:text.index(last, start)]


def orders(text, tiles=12, stages=2):
    """Edges a -> b, "a is over before b starts", of the walk as the source has it, and the ring that each row's term comes with."""
    producer = section(text, "if (warp == 8) {", "} else if (warp == 9) {")
    issuer = section(text, "for (int u = 0; u < total && ok; ++u) {", "if (ok && total > 0) commit_by(leader, acc_full);")
    rows = section(text, "const float *rows = reinterpret_cast<const float *>(smem + L::OFF_ROWS", "hand_over(p, dp_at, ds_ready);")
    # the ring that brings each term: the `load` that is given it, or is told (true) to bring both
    calls = re.findall(r"load\((q|g)_full, ([^()]*)\)", producer)
    ring = {term: next(name for name, rest in calls if f"P.row_{term}" in rest or " true," in rest) for term in ("lse", "delta")}
    # what the issuing warp does in an iteration, in its order
    steps = re.findall(r"warp_wait\((p_ready|ds_ready)|product_tokens\(leader, (DV|DK)|commit_by\(leader, &(q|g)_empty", issuer)
    steps = [next(x for x in s if x) for s in steps]
    released_after = {}   # ring -> the row warps' arrivals that its release comes after
    waited = []
    for s in steps:
        if s in ("p_ready", "ds_ready"):
            waited.append(s)
        elif s in ("q", "g"):
            released_after[s] = list(waited)
    # where the row warps read the terms: before or after they say that P is there
    read_before = {"lse": "p_ready" if rows.index("rows + 8 * i") < rows.index("p_ready") else "ds_ready",
                   "delta": "p_ready" if rows.index("rows + TILE + 8 * i") < rows.index("hand_over(p, s_at, p_ready)") else "ds_ready"}
    edges = {}

    def edge(a, b):
        edges.setdefault(a, set()).add(b)

    for u in range(tiles):
        for term in ("lse", "delta"):
            edge(("read", term, u), (read_before[term], u))
        for name in ("q", "g"):
            for arrival in released_after[name]:
                edge((arrival, u), ("empty", name, u))
            edge(("empty", name, u), ("copy", name, u + stages))
        edge(("p_ready", u), ("ds_ready", u))           # a row warp's own order
        edge(("ds_ready", u), ("read", "lse", u + 1))
    return edges, ring


def reaches(edges, a, b):
    todo, seen = [a], set()
    while todo:
        at = todo.pop()
        if at == b:
            return True
        for x in edges.get(at, ()):
            if x not in seen:
                seen.add(x)
                todo.append(x)
    return False


@pytest.mark.parametrize("stages", [2, 4])
@pytest.mark.parametrize("term", ["lse", "delta"])
def test_a_tile_s_row_terms_are_read_before_their_stage_is_written_anew(term, stages):
    edges, ring = orders(keys_walk(), stages=stages)
    for u in range(4):
        assert reaches(edges, ("read", term, u), ("copy", ring[term], u + stages)), \
            f"{term} of tile {u} may still be read when tile {u + stages} is copied over it (it comes with ring {ring[term]})"


@pytest.mark.parametrize("name", ["attention_forward.cu", "attention_backward.cu", "attention_parts.cu"])
def test_what_is_drained_after_a_wait_that_gave_up_is_committed_by_the_lane_that_issued_it(name):
    """A commit covers what its own thread issued.  The products are issued by the elected lane, so the commit behind which tensor memory is given back
    must be the elected lane's too, whichever that is."""
    text = (SOURCE.parent / name).read_text()
    issued = re.findall(r"(?:product_features<BLOCKS>|product_tokens(?:<\d, \d>)?|parts_along_\w+)\((\w+),", text)
    assert issued and set(issued) <= {"leader", "uint32_t"}, issued
    assert re.search(r"leader = elect_lane\(\)", text)
    drains = re.findall(r"if \([^;{}]*?\*abort_flag[^;{}]*?\) \{[^{}]*?drained[^{}]*?\}", text)
    assert len(drains) == (1 if name == "attention_forward.cu" else 2)
    for block in drains:
        assert "commit_by(elect_lane()," in block and "tc_commit" not in block and "lane == 0" not in block, block


def test_no_barrier_of_the_queries_walk_is_two_phases_ahead_of_a_waiting_warp():
    """A wait by parity cannot tell a phase from the one two later.  So the phase that next completes on a barrier must depend on every warp having
    passed its wait for the one before: of the barriers that tiles take in turn, from the order of both roles in the source."""
    text = SOURCE.read_text()
    text = text[text.index("void queries_walk("):text.index("// Both walks in one launch")]
    issuer = section(text, "if (total > 0 && ok) ok = first(0);", "if (ok && total > 0) commit_by(leader, acc_full);")
    first = section(text, "auto first = [&](int u) {", "return true;\n        };")
    rows = section(text, "const bool masked = j0 < all_lo", "if (ok && total > 0) {\n            ok = warp_wait(acc_full")

    def ops(code):
        """(what, barrier, tile offset) in the order of the source."""
        found = []
        for m in re.finditer(r"warp_wait\(&?(\w+)|commit_by\(leader, &?(\w+)|mbar_arrive\(&?(\w+)|\bfirst\(u \+ 1\)", code):
            wait, commit, arrive = m.groups()
            found.append(("wait", wait, 0) if wait else ("arrive", commit or arrive, 0) if commit or arrive else ("first", None, 1))
        return found

    barriers = ("s_full", "s_read", "dp_full", "ds_ready")
    # tiles take one barrier, or two in turn where the source picks it by the tile's last bit
    count = {b: 2 if re.search(rf"&{b}\[u & 1\]", rows) else 1 for b in barriers}
    assert all(("wait", b, 0) in ops(issuer) + ops(first) + ops(rows) for b in barriers)
    edges, tiles = {}, 12

    def chain(sequence):
        for a, b in zip(sequence, sequence[1:]):
            edges.setdefault(a, set()).add(b)

    issued = [(w, b, 0) for w, b, _ in ops(first)]
    for u in range(tiles):
        for w, b, at in ops(issuer):
            issued += [(x, y, u + 1) for x, y, _ in ops(first)] if w == "first" else [(w, b, u)]
    chain(issued)
    chain([(w, b, u) for u in range(tiles) for w, b, _ in ops(rows)])
    for b in barriers:
        for u in range(tiles):
            edges.setdefault(("arrive", b, u), set()).add(("wait", b, u))
    for b in barriers:
        for u in range(4):
            assert reaches(edges, ("wait", b, u), ("arrive", b, u + count[b])), \
                f"{b}: tile {u + count[b]} may arrive before a warp has seen that tile {u} has"


def test_products_of_the_float32_walks_wait_for_the_tiles_they_read():
    """Two warps issue the products of a walk.  Each tile that a product reads has arrived: its issuing warp waited for it, or for something that was made of it."""
    text = (SOURCE.parent / "attention_parts.cu").read_text()
    text = section(text, "if (OF_KEYS && warp == 9) {   // S, dV", "if (ok && total > 0) commit_by(leader, bar.all_full);")
    branches = [text[:text.index("} else if (OF_KEYS) {")], text[text.index("} else if (OF_KEYS) {"):text.index("} else if (warp == 9) {")],
                text[text.index("} else if (warp == 9) {"):text.index("} else {   // dP")]]
    # The row warps of dK's gradients wait for the scores (ring x) and for dP, so x has arrived where they say that these are ready.  The row warps of dV's
    # probabilities wait for the scores alone, which says nothing of ring y.
    implied = {"p_ready": "", "ds_ready": "x"}
    for branch, ring in zip(branches, ("y", "x", "x")):
        loop = branch[branch.index("for (int u = 0;"):]
        before = loop[:loop.index("sums(SUM")]
        assert re.search(rf"ring_{ring} \+ \(u %", loop[loop.index("sums(SUM"):])
        own = f"arrived(bar.{ring}_full, u," in before or f"from_{ring}(u)" in branch or f"from_{ring}(u + 1)" in branch
        made = any(ring in implied[b] for b in re.findall(r"bar\.(p_ready|ds_ready)", before))
        assert own or made, f"the products that read ring {ring} do not wait for it:\n{branch}"
