"""CPU model of the barrier protocol of the adapter GEMM (wan2-ti2v-5b_b200/csrc/gemm.cu, kLoraRuns) and of its
down-projection (lora.cu): a ring of loads, sums over runs of stages in two accumulators in turn, and an
epilogue that adds the runs up while the next one is multiplied."""
import random

import pytest

from test_attn_protocol import Bar, _drive


def run(tiles, ring, stages_a_run, seed, checked=True):
    """tiles: [(K blocks, adapter stages)].  Returns the tiles as the epilogue saw them: [[stages of each run]]."""
    rnd = random.Random(seed)
    full, empty = [Bar(1) for _ in range(ring)], [Bar(1) for _ in range(ring)]
    u_req, u_ok = [Bar(1) for _ in range(ring)], [Bar(2) for _ in range(ring)]
    tfull, tempty = [Bar(2) for _ in range(2)], [Bar(1) for _ in range(2)]
    said, holds = [None, None], [None] * ring
    acc_holds, pipe, seen, wrong = [[], []], [], [], []

    def producer():
        n = 0
        for t, (kb, ad) in enumerate(tiles):
            for i in range(kb + ad):
                yield ("wait", empty[n % ring], (n // ring & 1) ^ 1)
                if checked and i >= kb:
                    u_req[n % ring].arrive()
                yield ("work", rnd.randint(1, 4))
                holds[n % ring] = (t, i)
                full[n % ring].arrive()
                n += 1

    def issuer():
        n = acc = ph = 0
        ok = [0] * ring
        for t, (kb, ad) in enumerate(tiles):
            used = 0
            yield ("wait", tempty[acc], ph ^ 1)
            acc_holds[acc] = []
            for i in range(kb + ad):
                if used == stages_a_run:
                    said[acc] = False
                    tfull[acc].arrive()
                    pipe.append(["commit", tfull[acc]])
                    acc ^= 1
                    ph ^= acc == 0
                    used = 0
                    yield ("wait", tempty[acc], ph ^ 1)
                    acc_holds[acc] = []
                yield ("wait", full[n % ring], n // ring & 1)
                if holds[n % ring] != (t, i):
                    wrong.append((t, i))
                if checked and i >= kb:
                    yield ("wait", u_ok[n % ring], ok[n % ring])
                    ok[n % ring] ^= 1
                acc_holds[acc].append((t, i))
                pipe.append(["mma", rnd.randint(1, 3)])
                pipe.append(["commit", empty[n % ring]])
                used += 1
                n += 1
            said[acc] = True
            tfull[acc].arrive()
            pipe.append(["commit", tfull[acc]])
            acc ^= 1
            ph ^= acc == 0

    def check():
        n, req = 0, [0] * ring
        for t, (kb, ad) in enumerate(tiles):
            n += kb
            for i in range(ad):
                yield ("wait", u_req[n % ring], req[n % ring])
                yield ("wait", full[n % ring], n // ring & 1)
                if holds[n % ring] != (t, kb + i):
                    wrong.append(("check", t, i))
                req[n % ring] ^= 1
                yield ("work", rnd.randint(1, 3))
                u_ok[n % ring].arrive()
                n += 1

    def epilogue():
        acc = ph = 0
        for _ in tiles:
            runs = []
            while True:
                yield ("wait", tfull[acc], ph)
                last, at = said[acc], list(acc_holds[acc])
                runs.append(at)
                yield ("work", rnd.randint(1, 9 if not last else 30))  # the last one is kept over the tile's epilogue
                if acc_holds[acc] != at:
                    wrong.append(("overwritten", at))
                tempty[acc].arrive()
                acc ^= 1
                ph ^= acc == 0
                if last:
                    break
            seen.append(runs)

    agents = {"p": producer(), "i": issuer(), "e": epilogue()}
    if checked:
        agents |= {"c0": check(), "c1": check()}
    assert _drive(agents, pipe, rnd), "the roles wait for one another"
    assert not wrong, wrong[:3]
    return seen


@pytest.mark.parametrize("ring", [4, 5, 6])
def test_runs_of_the_adapter_gemm(ring):
    for seed in range(60):
        rnd = random.Random(1000 + seed)
        tiles = [(rnd.choice([1, 2, 7, 8, 9, 16, 30]), rnd.choice([0, 3, 6, 12])) for _ in range(rnd.randint(1, 5))]
        seen = run(tiles, ring, 8, seed)
        for t, (kb, ad) in enumerate(tiles):
            assert [i for r in seen[t] for i in r] == [(t, i) for i in range(kb + ad)]  # each stage once, in order
            assert all(len(r) == 8 for r in seen[t][:-1]) and 0 < len(seen[t][-1]) <= 8


def test_runs_of_the_down_projection():
    """Passes in place of tiles; no stage is looked through."""
    for seed in range(60):
        rnd = random.Random(2000 + seed)
        kb = rnd.randint(1, 40)
        run([(kb, 0)] * rnd.randint(1, 4), 4, 8, seed, checked=False)
