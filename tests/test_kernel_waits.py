"""Rules of the barrier waits in the pipelined layer kernels, read from their source (a wait that goes wrong shows on a
device only as a hang, so it is looked for here).

A bounded wait may give up in one lane and succeed in its neighbour.  Where a whole warp waits, the lanes therefore agree
on the result before they act on it: those that left alone would stay away from the warp-wide instructions that follow."""
from __future__ import annotations

import random
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "draw-instant_b200" / "csrc"
KERNELS = [("k_xattn.cu", "xattn_kernel"), ("k_lora.cu", "lora_t_kernel"), ("k_lora.cu", "lora_tile_kernel"),
           ("k_lora.cu", "list_adapters")]
WAIT = re.compile(r"\b(?:wait_on|mbar_wait)(?:<\w+>)?\(")


def closing(text, at):
    """Index of the brace that closes the one at `at`."""
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return i
    raise AssertionError("unbalanced braces")


def body(file, name):
    """A function's text, without comments."""
    text = re.sub(r"/\*.*?\*/|//[^\n]*", "", (CSRC / file).read_text(), flags=re.S)
    m = re.search(r"__(?:launch_bounds__\([^{;]*\)|forceinline__)[^{;]*\b%s\([^{;]*\) \{" % name, text)
    assert m, f"{file}: no {name}"
    return text[m.end() - 1:closing(text, m.end() - 1) + 1]


def one_thread(text):
    """Spans that a single thread of a warp runs."""
    heads = re.finditer(r"if \((?:[^;{}]*\belect_one\(\)|lane == 0|threadIdx\.x == 0)\) \{", text)
    return [(m.start(), closing(text, m.end() - 1)) for m in heads]


def inside(spans, at):
    return any(a <= at <= b for a, b in spans)


def statement(text, at):
    """The statement around `at`, and the one behind it."""
    start = max(text.rfind(c, 0, at) for c in ";{}") + 1
    end = text.index(";", at)
    return text[start:end].strip(), text[end + 1:text.index(";", end + 1)].strip()


def unagreed(text):
    """Waits of a whole warp whose lanes may go on with different results."""
    alone = one_thread(text)
    lambdas = [(m.group(1), m.start(), closing(text, m.end() - 1))
               for m in re.finditer(r"auto (\w+) = \[&\](?:\([^{;]*?\))?(?: -> [\w ]+\*)? \{", text)]
    bad = []
    for m in WAIT.finditer(text):
        if inside(alone, m.start()):
            continue
        now, then = statement(text, m.start())
        if "__all_sync(" in now or WAIT.match(now):  # agreed on at once, or a wait whose result is dropped
            continue
        var = re.match(r"(?:const )?(?:bool )?(\w+) = ", now)
        if var and re.search(r"__all_sync\(0xffffffffu, %s\)" % var.group(1), then):
            continue
        around = [n for n, a, b in lambdas if a <= m.start() <= b]
        calls = [c.start() for n in around for c in re.finditer(r"(?<![.\w])%s\(" % n, text)]
        if calls and all(inside(alone, c) for c in calls):  # a helper of single threads
            continue
        bad.append(now)
    return bad


@pytest.mark.parametrize("file,name", KERNELS)
def test_a_warps_lanes_agree_on_a_wait(file, name):
    text = body(file, name)
    assert len(WAIT.findall(text)) > 0
    assert unagreed(text) == []


# barriers on which a warp gives back the entry of a list or of the items that it has read
PLACES = re.compile(r"if \((?:any && )?lane == 0\) mbar_arrive(?:_relaxed)?\(&(?:item_empty|list_empty|o_read|d_empty|list_full)\[[^]]*\]\)")


def early_releases(text):
    """Places where lane 0 gives an entry back before the other lanes' reads of it are over."""
    alone = [s for s in one_thread(text) if not text.startswith("if (lane == 0)", s[0])]
    bad = []
    for m in PLACES.finditer(text):
        if not inside(alone, m.start()) and not re.search(r"__syncwarp\(\);\s*$", text[:m.start()]):
            bad.append(m.group(0))
    for m in re.finditer(r"if \(lane == 0\) \{", text):
        block = text[m.end():closing(text, m.end() - 1)]
        if re.search(r"_empty\[", block) and not re.search(r"__syncwarp\(\);\s*$", text[:m.start()]):
            bad.append(block.strip())
    return bad


@pytest.mark.parametrize("file,name", KERNELS)
def test_a_warp_has_read_what_its_first_lane_gives_back(file, name):
    """What follows a release may overwrite the entry at once; only a warp barrier orders the other lanes' reads before it."""
    text = body(file, name)
    assert PLACES.search(text)
    assert early_releases(text) == []


# ---- the ring of key and value tiles --------------------------------------------------------------------------

class Barrier:
    def __init__(self, count):
        self.count, self.left, self.done = count, count, 0  # done: phases completed

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.done = self.count, self.done + 1

    def passed(self, parity):
        return (self.done - 1) % 2 == parity


def ring_roles(ring, tiles, masked, counts, cleaner_arrives):
    """Loader, MMA and cleaning warp of one CTA as generators that yield while they wait; the i-th tile is a K tile for even
    i and a V tile for odd i.  A tile that is refilled before the cleaning warp has seen it is an error."""
    full, empty, clean = ([Barrier(n) for _ in range(ring)] for n in counts)
    holds, seen = [None] * ring, set()

    def loader():
        for i in range(tiles):
            s = i % ring
            while not empty[s].passed((i // ring) % 2 ^ 1):
                yield
            assert i < ring or i - ring in seen, "refilled unseen"
            holds[s] = i
            full[s].arrive()
            yield

    def mma():
        cleaned = [0] * ring
        for i in range(tiles):
            s = i % ring
            while not full[s].passed((i // ring) % 2):
                yield
            if i % 2 and masked[i // 2]:
                while not clean[s].passed(cleaned[s]):
                    yield
                cleaned[s] ^= 1
            assert holds[s] == i
            empty[s].arrive()
            yield

    def cleaner():
        for i in range(tiles):
            s = i % ring
            while not full[s].passed((i // ring) % 2):
                yield
            assert holds[s] == i, "another tile"
            seen.add(i)
            if i % 2 and masked[i // 2]:
                clean[s].arrive()
            if cleaner_arrives:
                empty[s].arrive()
            yield

    return {"loader": loader(), "mma": mma(), "cleaner": cleaner()}


@pytest.mark.parametrize("slow", ["none", "loader", "mma", "cleaner"])
@pytest.mark.parametrize("ring", [4, 5, 6, 7, 10])
def test_no_tile_is_refilled_before_every_role_has_seen_it(ring, slow):
    """The barriers with the kernel's own arrival counts, under schedules that hold one role back as long as they can."""
    text = body("k_xattn.cu", "xattn_kernel")
    counts = [int(re.search(r"mbar_init\(&%s\[i\], (\d+)\)" % b, text).group(1)) for b in ("kv_full", "kv_empty", "v_clean")]
    at = text.index("{", text.index("if (svc == 2)"))
    arrives = "&kv_empty[" in text[at:closing(text, at)]
    rng = random.Random(ring)
    for share in (0.0, 0.3, 1.0):
        masked = [rng.random() < share for _ in range(40)]
        roles = ring_roles(ring, 2 * len(masked), masked, counts, arrives)
        idle = 0
        while roles:
            assert idle < 2000, "roles wait for one another"
            fast = [r for r in roles if r != slow] if idle < 30 else list(roles)  # the slow one only when nothing else moves
            name = rng.choice(fast or list(roles))
            before = roles[name].gi_frame.f_locals.get("i")
            try:
                next(roles[name])
                idle = 0 if roles[name].gi_frame.f_locals.get("i") != before else idle + 1
            except StopIteration:
                del roles[name]
                idle = 0
