"""Recipes of the documentation, run on the CPU: their calls go to an engine that only keeps the rows that they would write."""
import re
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

ROOT = Path(__file__).resolve().parents[1]
PREFIX, SLOT, B, ROOM = 8192, 2, 4, 1 << 15


def recipes():
    """Every Python block that decodes over a shared prefix, and the blocks of its section behind it."""
    found = []
    for page in sorted(ROOT.glob("*.md")):
        for section in re.split(r"^##+ ", page.read_text(), flags=re.M):
            blocks = re.findall(r"```python\n(.*?)```", section, flags=re.S)
            if blocks and "decode_prefix_device(" in blocks[0]:
                found.append(blocks)
    return found


class Rows:
    """The K/V rows of every sequence as the numbers of the tokens that they hold, and the calls that write or move them."""

    def __init__(self, names):
        self.names = names  # the recipe's own, its tensors among them
        self.rows = [list(range(PREFIX)) if b == SLOT else [] for b in range(B)]
        self.steps = 0

    def tensor(self, ptr):
        return next(t for t in self.names.values() if torch.is_tensor(t) and t.data_ptr() == ptr)

    def of(self, ptr):
        return self.tensor(ptr).tolist()

    def qk_norm_rotary_device(self, *args, b, **kw):
        pass

    def qk_norm_rotary_step_device(self, qkv, ld, wq, wk, positions, q, form, *, rows_ptr):
        for b, (p, t) in enumerate(zip(self.of(positions), self.of(rows_ptr))):
            if p >= 0 and 0 <= t < ROOM:
                self.rows[b][t:t + 1] = [p]
        self.steps += 1

    def decode_prefix_device(self, q, slot, prefix_len, lens, o, **kw):
        assert slot == SLOT and prefix_len == PREFIX
        assert self.rows[SLOT][:PREFIX] == list(range(PREFIX)), "the prefix's rows were written over or moved"
        assert all(n == len(r) for b, (n, r) in enumerate(zip(self.of(lens), self.rows)) if b != SLOT)

    def attention_mass_step_device(self, q, lens, lse, mass, **kw):
        pass

    def evict_device(self, mass, lens, keep, kept, *, sinks, recent):
        for b, n in enumerate(self.of(lens)):
            if n > keep:
                self.rows[b] = self.rows[b][:keep - recent] + self.rows[b][n - recent:n]
                self.tensor(lens)[b] = keep


@pytest.mark.parametrize("goes_on", [False, True])
def test_a_shared_prefix_stays_what_it_is(goes_on):
    """Steps and evictions as the recipe has them leave the rows that all sequences attend alone, also where the slot that
    holds them goes on itself."""
    (first, *rest), = recipes()
    prompt, step = first.split("# each step", 1)
    step, evict = step.split("# every so often", 1)
    lens = torch.zeros(B, dtype=torch.int32)
    positions = torch.full((B,), PREFIX, dtype=torch.int32)
    names = dict(lens=lens, positions=positions, mass=torch.zeros(1), system_slot=SLOT, prefix_len=PREFIX, n=PREFIX, ld=0,
                 lens_ptr=lens.data_ptr(), positions_ptr=positions.data_ptr())
    names.update({f"{t}_ptr": 0 for t in ("qkv", "q", "o", "lse", "kept", "mass")})
    acc = names["acc"] = Rows(names)

    exec(prompt, names)
    if goes_on:
        lens[SLOT] = positions[SLOT] = PREFIX
        evict, = rest
    for i in range(3000):
        exec("#" + step, names)
        if i % 1000 == 999:
            exec("#" + evict if not goes_on else evict, names)
            assert lens.tolist() == [0 if b == SLOT and not goes_on else len(r) for b, r in enumerate(acc.rows)]
    assert acc.steps == 3000 and int(lens[0]) < 3000 and len(acc.rows[SLOT]) == PREFIX + (3000 if goes_on else 0)
