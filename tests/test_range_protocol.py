"""CPU model of the barrier protocol of range_attn_kernel (wan2-ti2v-5b_b200/csrc/attn_range.cu).

On top of the unmasked attention's protocol (test_attn_protocol.py) come a queue of units, query
tiles of a pair that skip key tiles, and two warps that look through the V tiles which are not seen
by every row before they are multiplied.  The model also notes which load a ring slot holds, so a
wait that passes a phase too early shows as a wrong load."""
import os
import random
import re

from test_attn_protocol import Bar, _drive


def run(units, ring, seed, announced=True):
    """units: [(ranges of tile 0, of tile 1, partial key tiles)], ranges as (first, end) key tiles."""
    rnd = random.Random(seed)
    kv_full, kv_empty = [Bar(1) for _ in range(ring)], [Bar(1) for _ in range(ring)]
    v_ok, v_req = [Bar(2) for _ in range(ring)], [Bar(1) for _ in range(ring)]
    q_full, q_empty = Bar(1), Bar(1)
    s_full, p_part, p_full, o_done = ([Bar(1) for _ in range(2)] for _ in range(4))
    u_full, u_empty = [Bar(1) for _ in range(2)], [Bar(5) for _ in range(2)]  # MMA, 2 softmax groups, 2 checks
    holds = [None] * ring
    pipe, wrong = [], []

    def has(u, t, j):
        return u[t][0] <= j < u[t][1]

    def tiles(u):
        ends = [r for r in u[:2] if r[0] < r[1]]
        return [j for j in range(min(r[0] for r in ends), max(r[1] for r in ends)) if has(u, 0, j) or has(u, 1, j)] \
            if ends else []

    def producer():
        g = q = 0
        for i in range(len(units) + 1):
            yield ("wait", u_empty[i % 2], (i // 2 & 1) ^ 1)
            u_full[i % 2].arrive()
            if i == len(units):
                return
            js = tiles(units[i])
            if not js:
                continue
            yield ("wait", q_empty, (q & 1) ^ 1)
            q += 1
            yield ("work", rnd.randint(1, 4))
            q_full.arrive()
            for j in js:
                for x in "KV":
                    yield ("wait", kv_empty[g % ring], (g // ring & 1) ^ 1)
                    if x == "V" and j in units[i][2]:
                        v_req[g % ring].arrive()
                    yield ("work", rnd.randint(1, 5))
                    holds[g % ring] = (i, j, x)
                    kv_full[g % ring].arrive()
                    g += 1

    def issuer():
        g = q = 0
        np, ok = [0, 0], [0] * ring
        for i in range(len(units) + 1):
            yield ("wait", u_full[i % 2], i // 2 & 1)
            if i == len(units):
                return
            u_empty[i % 2].arrive()
            u = units[i]
            js = tiles(u)
            if not js:
                continue

            def kv(r, j, x):
                yield ("wait", kv_full[r % ring], r // ring & 1)
                if holds[r % ring] != (i, j, x):
                    wrong.append(("mma", i, j, x))

            def qk(t):
                pipe.append(["mma", rnd.randint(2, 4)])
                pipe.append(["commit", s_full[t]])

            def pv(t, j):
                ph = np[t] & 1
                np[t] += 1
                yield ("wait", p_part[t], ph)
                pipe.append(["mma", rnd.randint(1, 3)])
                yield ("wait", p_full[t], ph)
                pipe.append(["mma", rnd.randint(1, 2)])
                if j == u[t][1] - 1:
                    pipe.append(["commit", o_done[t]])

            yield ("wait", q_full, q & 1)
            q += 1
            yield from kv(g, js[0], "K")
            for t in (0, 1):
                if has(u, t, js[0]):
                    qk(t)
            pipe.append(["commit", kv_empty[g % ring]])
            if len(js) == 1:
                pipe.append(["commit", q_empty])
            for n, j in enumerate(js):
                nxt = js[n + 1] if n + 1 < len(js) else None
                vs, ks = (g + 1) % ring, (g + 2) % ring
                yield from kv(g + 1, j, "V")
                if j in u[2]:
                    yield ("wait", v_ok[vs], ok[vs])
                    ok[vs] ^= 1
                if has(u, 0, j):
                    yield from pv(0, j)
                if nxt is not None:
                    yield from kv(g + 2, nxt, "K")
                    if has(u, 0, nxt):
                        qk(0)
                if has(u, 1, j):
                    yield from pv(1, j)
                pipe.append(["commit", kv_empty[vs]])
                g += 2
                if nxt is None:
                    break
                if has(u, 1, nxt):
                    qk(1)
                pipe.append(["commit", kv_empty[ks]])
                if n + 2 == len(js):
                    pipe.append(["commit", q_empty])

    def check():
        g, req = 0, [0] * ring
        for i in range(len(units) + 1):
            yield ("wait", u_full[i % 2], i // 2 & 1)
            if i == len(units):
                return
            u_empty[i % 2].arrive()
            for j in tiles(units[i]):
                r = g + 1
                if j in units[i][2]:
                    if announced:
                        yield ("wait", v_req[r % ring], req[r % ring])
                        req[r % ring] ^= 1
                    yield ("wait", kv_full[r % ring], r // ring & 1)
                    if holds[r % ring] != (i, j, "V"):
                        wrong.append(("check", i, j))
                    yield ("work", rnd.choice([1, 3, 8, 60]))  # slow at times: the others must not run away
                    v_ok[r % ring].arrive()
                g += 2

    def softmax(t):
        g = ns = no = 0
        ok = [0] * ring
        for i in range(len(units) + 1):
            yield ("wait", u_full[i % 2], i // 2 & 1)
            if i == len(units):
                return
            u_empty[i % 2].arrive()
            u, any_tile = units[i], False
            for j in tiles(u):
                vs = (g + 1) % ring
                g += 2
                if not has(u, t, j):
                    if j in u[2]:
                        ok[vs] ^= 1
                    continue
                any_tile = True
                yield ("wait", s_full[t], ns & 1)
                ns += 1
                yield ("work", rnd.randint(1, 6))
                if j in u[2]:
                    yield ("wait", v_ok[vs], ok[vs])
                    ok[vs] ^= 1
                    if holds[vs] != (i, j, "V"):
                        wrong.append(("softmax", i, j))
                yield ("work", rnd.randint(1, 6))
                p_part[t].arrive()
                yield ("work", rnd.randint(1, 3))
                p_full[t].arrive()
            if any_tile:
                yield ("wait", o_done[t], no & 1)
                no += 1
            yield ("work", rnd.randint(1, 6))

    agents = {"producer": producer(), "issuer": issuer(), "check0": check(), "check1": check(), "softmax0": softmax(0),
              "softmax1": softmax(1)}
    return _drive(agents, pipe, rnd) and not wrong


def random_units(rnd):
    units = []
    for _ in range(rnd.randint(1, 6)):
        r = []
        for _ in range(2):
            a = rnd.randint(0, 12)
            r.append((a, a + rnd.choice([0, 1, 1, 2, 5, 9, 14])))
        units.append((*r, {j for j in range(30) if rnd.random() < rnd.choice([0.1, 0.5, 1.0])}))
    return units


def test_range_protocol_never_deadlocks():
    for seed in range(120):
        units = random_units(random.Random(seed))
        for ring in (5, 8):  # head_dim 128 and 64
            assert run(units, ring, seed), (units, ring, seed)


def test_tiles_to_check_must_be_announced():
    """Waiting for the load alone lets a checking warp run ahead of the ring by two phases of a slot:
    it then reads an older load, and the protocol can stop."""
    fails = 0
    for seed in range(60):
        rnd = random.Random(seed)
        units = [((0, 20), (0, 20), {19}) for _ in range(rnd.randint(1, 4))]
        fails += not run(units, 5, seed, announced=False)
    assert fails > 0


def test_what_the_launch_before_writes_is_read_with_plain_loads():
    """The tile attention and the adapter GEMM start beside the launch that plans for them.  The read-only path
    is for memory that stays as it is over the whole kernel, so it may read a call's inputs only."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wan2-ti2v-5b_b200", "csrc")
    inputs = {
        "attn_range.cu": {"a.lo", "a.hi", "a.pos", "a.slopes", "a.table", "p.a.table", "a.q"},
        "lora.cu": {"a.ids", "a.scales", "xp", "dp", "x0", "x1", "up"},
        "gemm.cu": {"a.bias", "a.gate_mod", "a.gate_e0", "gate_row", "lo->ids", "bp", "mp", "ep"},
    }
    for name, allowed in inputs.items():
        with open(os.path.join(csrc, name)) as f:
            read = re.findall(r"__ldg\((?:reinterpret_cast<[^>]*>\()?\s*([\w.>-]+)", f.read())
        assert read and not set(read) - allowed, (name, set(read) - allowed)
