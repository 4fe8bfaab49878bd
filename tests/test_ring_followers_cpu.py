"""The CTA-pair GEMM's ring, roles that put nothing into an expand step's slot (the block scales' producer and the scale copiers of an
FP4 base): a model of the ring's barriers run under every role's worst delay.  A parity wait says "the phase in progress is not of
this parity", so a role that follows a barrier without taking part in it, and comes two phases late, waits for good.  The model takes
from the kernel's source how each role treats such a slot."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parent.parent / "onebase_b200" / "csrc" / "k2_prefill2.cu"
STAGES = 5


def passes_steps_by(where: int) -> bool:
    """Whether the loop whose slot wait is numbered `where` waits only in k-block slots, behind the producer's `k_free`."""
    text = SOURCE.read_text()
    at = text.index(f"limit_ns, {where}, it)")
    body = text[text.rindex("for (int q = 0", 0, at): at]
    return re.search(r"if \(!step\) \{|if \(step\) \{\s*last_step = it;\s*\} else \{", body) is not None and "&ctrl->k_free[st]" in body


class Barrier:
    """One mbarrier: completed phases; `parts` of the phase in progress still to come (set when the phase is opened)."""

    def __init__(self):
        self.done = 0
        self.got = set()

    def passed(self, parity: int) -> bool:
        return (self.done & 1) != parity

    def arrive(self, who: str, need: set):
        self.got.add(who)
        if self.got >= need:
            self.got = set()
            self.done += 1


def ring(tiles, by_scales: bool, by_copier: bool):
    """Generators of the roles; each yields a predicate to wait for.  `tiles`: per tile the slots, True = expand step."""
    full, sf, empty, k_free = ([Barrier() for _ in range(STAGES)] for _ in range(4))
    slots = [step for t in tiles for step in t]

    def producer():
        for it, step in enumerate(slots):
            st, ph = it % STAGES, (it // STAGES + 1) & 1
            yield lambda: empty[st].passed(ph)
            if not step:
                k_free[st].arrive("producer", {"producer"})
            full[st].arrive("data", {"data"} if step else {"data", "scales"})

    def scales(by: bool):
        uses = [0] * STAGES
        for it, step in enumerate(slots):
            st, use = it % STAGES, it // STAGES
            if not by:
                yield lambda: empty[st].passed((use + 1) & 1)
            elif not step:
                yield lambda: k_free[st].passed(uses[st] & 1)
                uses[st] += 1
            if not step:
                give_scales(st, use)

    def copier(by: bool):
        uses, last = [0] * STAGES, -STAGES - 1
        for it, step in enumerate(slots):
            st, use = it % STAGES, it // STAGES
            if step:
                last = it
                if by:
                    continue
            elif by:
                if it - last <= STAGES:
                    yield lambda: k_free[st].passed(uses[st] & 1)
                uses[st] += 1
            yield lambda: full[st].passed(use & 1)
            if not step:
                copy(st, use)

    def give_scales(st, use):
        assert empty[st].done >= use, "scales into a slot that is not free"
        full[st].arrive("scales", {"data", "scales"})

    def copy(st, use):
        assert full[st].done > use, "scales copied before they landed"
        sf[st].arrive("copy", {"copy"})

    def issuer():
        seen = [0] * STAGES
        for it, step in enumerate(slots):
            st, use = it % STAGES, it // STAGES
            if step:
                yield lambda: full[st].passed(use & 1)
            else:
                yield lambda: sf[st].passed(seen[st] & 1)
                seen[st] += 1
            empty[st].arrive("mma", {"mma"})

    return {"producer": producer(), "scales": scales(by_scales), "copier": copier(by_copier), "issuer": issuer()}


def finishes(tiles, late: str, by_scales: bool, by_copier: bool) -> bool:
    """Runs the roles, `late` only when no other can move.  False: stuck."""
    roles = ring(tiles, by_scales, by_copier)
    waits = {n: next(r, None) for n, r in roles.items()}
    while any(w is not None for w in waits.values()):
        ready = [n for n, w in waits.items() if w is not None and w()]
        if not ready:
            return False
        n = next((m for m in ready if m != late), late)
        waits[n] = next(roles[n], None)
    return True


# k-blocks first, then steps (bf16 adapters); spread (stored ones, few k-blocks and many steps); none; one k-block
SHAPES = [[False] * 6 + [True] * 12, [False] * 5 + ([True] * 11 + [False]) * 3 + [True] * 7, [False] * 7, [False] + [True] * 512,
          [False] * 2 + [True] * 4, [False] * 3 + [True]]


@pytest.mark.parametrize("late", ["producer", "scales", "copier", "issuer"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_a_late_role_does_not_hang_the_ring(shape, late):
    tiles = [SHAPES[shape], SHAPES[(shape + 1) % len(SHAPES)], SHAPES[shape], SHAPES[2], SHAPES[shape]]
    assert finishes(tiles, late, passes_steps_by(21), passes_steps_by(13))


def test_the_model_shows_the_hazard():
    """Following a step's barriers without taking part in them: stuck once the role comes two phases late."""
    tiles = [SHAPES[0]] * 3
    assert not finishes(tiles, "scales", False, True) and not finishes(tiles, "copier", True, False)
