"""What a GPU test cannot show of the paged attention's kernels, checked in their sources. CPU only."""
import os
import re

from kore_b200.build import CSRC


def test_products_and_their_commits_are_one_threads():
    """tcgen05.commit follows the operations that the executing thread issued, and which lane elect.sync returns is not
    said: a commit by a fixed lane may follow nothing. So every product and every commit is issued under elect()."""
    with open(os.path.join(CSRC, "paged_tiles.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    body = text[text.index("MMA issuers") if "MMA issuers" in text else text.index("auto issuer ="):]
    calls = [m.start() for m in re.finditer(r"\b(?:commit|mma_ss<[^>]*>|mma_ts<[^>]*>)\(", body)]
    assert len(calls) >= 9
    guards = [m for m in re.finditer(r"if \(elect\(\)\)", body)]
    covered = []
    for g in guards:   # the statement or the block behind the guard
        at = g.end()
        while body[at].isspace():
            at += 1
        if body[at] != "{":
            covered.append((at, body.index(";", at)))
            continue
        depth, end = 0, at
        while True:
            depth += {"{": 1, "}": -1}.get(body[end], 0)
            if depth == 0:
                break
            end += 1
        covered.append((at, end))
    for c in calls:
        assert any(a <= c < b for a, b in covered), body[max(0, c - 60):c + 60]
