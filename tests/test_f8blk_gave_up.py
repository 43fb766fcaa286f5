"""Block-scaled e4m3 products whose bounded wait ran out store nothing, as the sources write them: a result with blocks of K missing would
look like any other.  The case cannot be made on a GPU without hanging it, so this reads the sources: each store of a result stands behind
a test of what the waits left."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paddock_b200", "csrc")


def kernel(name):
    """The kernel's body without comments."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    body = text[re.search(r"^f8blk_\w+_kernel\(", text, re.M).start():]
    return body[:body.index("\n}\n")]


def leaves_or_skips(text, at):
    """The conditions that decide whether the statement at `at` runs: of the blocks that enclose it, of its own statement, and of `if (..) return;`
    in front of it in the same blocks."""
    conditions, depth, i = [], 0, at
    start = max(text.rfind(c, 0, at) for c in ";{}") + 1
    conditions += re.findall(r"(?:if|for) (?:constexpr )?\(.*", text[start:at], re.S)
    while i > 0:
        i -= 1
        if text[i] == "}":
            depth += 1
        elif text[i] == "{":
            if depth:
                depth -= 1
                continue
            head = max(text.rfind(c, 0, i) for c in "{}") + 1
            conditions.append(text[head:i].split(";")[-1] if "for (" not in text[head:i] else text[head:i])
        elif depth == 0 and text.startswith("return;", i):
            conditions.append("return " + text[max(text.rfind(c, 0, i) for c in ";{}") + 1:i])
    return conditions


RESULTS = {"f8blk_split.cu": (r"\bstore_if\(out|\bstore4\(out|a\.hs\[[^;=]*\] = |\*reinterpret_cast<uint32_t\*>\(reinterpret_cast<uint8_t\*>\(a\.y\)", "gave_up", 8),
           "f8blk_wide.cu": (r"\bstore_row\(|\*reinterpret_cast<uint4\*>\(q|a\.hs\[[^;=]*\] = ", "ok", 3)}


@pytest.mark.parametrize("name", RESULTS)
def test_results_are_stored_only_where_no_wait_ran_out(name):
    pattern, word, least = RESULTS[name]
    body = kernel(name)
    found = list(re.finditer(pattern, body))
    assert len(found) >= least
    for m in found:
        conditions = leaves_or_skips(body, m.start())
        assert any(re.search(rf"\b{word}\b", c) for c in conditions), (m.group(), conditions)


def test_the_whole_cluster_hears_of_a_wait_that_ran_out():
    """The flag goes to every CTA of the cluster between its two meetings: behind the first all of them have set it to zero, behind the
    second all read it."""
    body = kernel("f8blk_split.cu")
    zeroed = body.index("sh->gave_up = 0;")
    first = body.index("cluster_sync();")
    told = body.index("&sh->gave_up")
    rest = [m.start() for m in re.finditer(r"cluster_sync\(\);", body)][1:]
    read = body.index("if (sh->gave_up")
    assert zeroed < first < told < rest[0] and all(any(r < m.start() for r in rest) for m in re.finditer(r"if \(sh->gave_up", body)) and read > rest[0]
    tell = body[max(body.rfind(c, 0, told) for c in ";{}"):told]
    assert "gave_up && threadIdx.x < split" in tell and "const bool gave_up = sh->abort_flag != 0;" in body[:told]


def test_both_halves_of_a_token_hear_of_a_wait_that_ran_out():
    """The gated front's scale is of both halves' warps: a half that gave up hands on NaN, and the other stores nothing either."""
    body = kernel("f8blk_wide.cu")
    handed = body.index("sh->amax[half][row] = ok ? m : __int_as_float(0x7fffffff);")
    taken = body.index("other = sh->amax[1u - half][row]")
    assert handed < body.index("bar.sync", handed) < taken < body.index("if (ok && other == other && t < a.batch)") < body.index("a.hs[")


@pytest.mark.parametrize("name", RESULTS)
def test_a_cta_that_gave_up_stays_until_its_copies_have_landed(name):
    """The role that gave up need not be the one with copies under way: the CTA waits, whoever it was, before it hands its shared memory on."""
    body = kernel(name)
    last = body.rindex("pdk_pdl_wait();")
    met = body.index("__syncthreads();", last)
    stays = re.search(r"if \(gave_up\) wait_for_copies\(\);|if \(sh->abort_flag\) wait_for_copies\(\);", body[met:])
    assert stays and "cluster_sync" not in body[met:met + stays.start()] and "tmem_dealloc" not in body[met:met + stays.start()]
    text = open(os.path.join(CSRC, "f8blk_tc5.cuh")).read()
    assert re.search(r"void wait_for_copies\(\) \{\s*for \(int i = 0; i < 64; \+\+i\) __nanosleep\(1000\);", text)
