"""How the warps of the attention kernels hand tiles to one another, on a model of their barriers (no GPU): whatever warp is late, every tile
is read in its own phase, nothing is overwritten while it is in use and every wait ends.  The numbers of arrivals come from the source."""
import os
import re

import pytest

from tests.ring_model import Bar, Meeting, Run

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nihilus_b200", "csrc")


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def _number(source, name, default=None):
    m = re.search(r"constexpr int %s\s*=\s*([0-9 +]+);" % name, source)
    return sum(int(x) for x in m.group(1).split("+")) if m else default


def _only_if_ok(source, arrival):
    """Whether every such arrival stands behind a condition on `ok`: a warp whose wait ran out makes none."""
    lines = source.splitlines()
    at = [i for i, line in enumerate(lines) if arrival in line]
    assert at, arrival
    return all("ok" in lines[i - 1] or "ok" in lines[i].split(arrival)[0] for i in at)


# ---- prompts: copies, products, two warps that watch the ring, sixteen of the softmax ----

KB = 1024


def _prompt_config(d, bf16, two):
    """(slots of the ring, score buffers) as attn_prompt.cu has them."""
    parts, buffers = (3, 2) if bf16 else (2, 3)
    queries = parts * (2 if two else 1) * 128 * d * 2
    return min(8, (224 * KB - queries) // (128 * d * 2)), buffers


CONFIGS = [(d, bf16, two) for d in (64, 128) for bf16 in (False, True) for two in (False, True) if not (bf16 and d == 128 and two)]


def k_at(j, ahead):
    return j + max(0, j - ahead + 1)


def v_at(j, n, ahead):
    return j + min(ahead + j, n)


def prompt_run(config, n, **schedule):
    """A CTA over n key tiles."""
    two = config[2]
    slots, buffers = _prompt_config(*config)
    source = _source("attn_prompt.cu")
    empty_arrivals = _number(source, "EMPTY_ARRIVALS", 1)
    careful = all(_only_if_ok(source, a) for a in ("mbar_arrive(&hd->p_full[buf])", "mbar_arrive(&hd->p_full[(2", "mbar_arrive_n(&hd->p_full["))
    drained, needed_only = "hd->drain" in source, "again(" in source
    run = Run(**schedule)
    ahead, steps = (buffers - 1, 2 * n) if two else (buffers, n)
    full, empty = [Bar(1) for _ in range(slots)], [Bar(empty_arrivals) for _ in range(slots)]
    s_full, p_full = [Bar(1) for _ in range(buffers)], [Bar(_number(source, "P_ARRIVALS")) for _ in range(buffers)]
    o_full, q_full = [Bar(1), Bar(1)], Bar(16)
    softmax, chains, end = Meeting(16), [Meeting(8), Meeting(8)], Meeting(20)
    drain = Bar(1)
    content, scores_of, product = [None] * slots, [None] * buffers, [None]
    untaken, left = [0], [0] * buffers  # warps that have yet to take the product; warps that have left their weights over the scores

    def land(slot, tile):
        content[slot] = tile

    def copies():
        kj = vj = issued = 0
        for at in range(2 * n):
            is_v = not (kj < n and kj < ahead + vj)
            tile = ("v", vj) if is_v else ("k", kj)
            kj, vj = kj + (not is_v), vj + is_v
            assert at == (v_at(tile[1], n, ahead) if is_v else k_at(tile[1], ahead))
            s = at % slots
            if not (yield empty[s], ((at // slots) & 1) ^ 1):
                break
            content[s] = None
            full[s].arrive(tx=1)
            run.copies.append((full[s], lambda s=s, tile=tile: land(s, tile)))
            issued += 1
        if drained:
            for at in range(max(0, issued - slots), issued):
                yield full[at % slots], (at // slots) & 1, True
        yield end, end.join()

    def use(slot, tile, t, buf, is_scores):
        run.check(content[slot] == tile, "a product reads", content[slot], "for", tile)
        if is_scores:
            scores_of[buf], left[buf] = t, 0
        else:
            run.check(scores_of[buf] == t and left[buf] == 8, "weights of", left[buf], "warps of", scores_of[buf], "for", t)
            run.check(untaken[0] == 0, "a product is overwritten")
            product[0], untaken[0] = t, 8

    def products():
        def issue(t, is_scores):
            j, buf = (t >> 1 if two else t), t % buffers
            at = k_at(j, ahead) if is_scores else v_at(j, n, ahead)
            s = at % slots
            run.products.append(lambda: use(s, ("k" if is_scores else "v", j), t, buf, is_scores))
            run.products.append(lambda: (s_full[buf] if is_scores else o_full[t & 1]).arrive())
            if (not two or t & 1) and not (needed_only and at + slots >= 2 * n):
                run.products.append(lambda: empty[s].arrive())

        ok = yield q_full, 0
        for t in range(min(buffers, steps)):
            if not ok:
                break
            at = k_at(t >> 1 if two else t, ahead)
            ok = yield full[at % slots], (at // slots) & 1
            if ok:
                issue(t, True)
        for t in range(steps):
            if not ok:
                break
            ok = yield p_full[t % buffers], (t // buffers) & 1
            if not ok:
                break
            issue(t, False)
            if t + buffers < steps:
                issue(t + buffers, True)
        if drained:
            run.products.append(drain.arrive)
            yield drain, 0, True
        yield end, end.join()

    def watcher(first):
        seen, ok = 0, True
        for t in range(steps):
            j = t >> 1 if two else t
            at = v_at(j, n, ahead)
            last = k_at((t + buffers) >> 1 if two else t + buffers, ahead) if t + buffers < steps else -1
            for target in (at, last):
                while seen <= target and ok:
                    ok = yield full[seen % slots], (seen // slots) & 1
                    if ok and empty_arrivals > 1:
                        empty[seen % slots].arrive()
                    seen += 1
                if target == at and ok:
                    run.check(content[at % slots] == ("v", j), "a watcher cleans", content[at % slots], "for", j)
            if t >= buffers and ok:
                ok = yield p_full[t % buffers], (t // buffers - 1) & 1
            if ok or not careful:
                p_full[t % buffers].arrive(1 + 8 if t == 0 and first else 1)
            if not ok:
                break
        yield end, end.join()

    def weights(chain):
        q_full.arrive()
        yield softmax, softmax.join()
        yield softmax, softmax.join()
        ok, use_ = True, 0
        for _ in range(0 if two else chain, n, 1 if two else 2):
            t = 2 * use_ + chain
            ok = ok and (yield s_full[t % buffers], (t // buffers) & 1)
            run.check(scores_of[t % buffers] == t, "scores", scores_of[t % buffers], "for", t)
            yield chains[chain], chains[chain].join()
            left[t % buffers] += 1
            yield None
            if ok or not careful:
                p_full[t % buffers].arrive()
            ok = ok and (yield o_full[chain], use_ & 1)
            run.check(product[0] == t, "product", product[0], "for", t)
            untaken[0] -= 1
            yield None
            if t + 1 < steps and (ok or not careful):
                p_full[(t + 1) % buffers].arrive()
            use_ += 1
        yield softmax, softmax.join()
        yield end, end.join()

    run.warps = {"copies of tiles": copies(), "products of tiles": products(), "watcher 2": watcher(True), "watcher 3": watcher(False)}
    for w in range(16):
        run.warps[f"softmax {w}"] = weights(w >> 3)
    run.go()


WARPS = ["copies of tiles", "products of tiles", "watcher 2", "watcher 3", "softmax 0", "softmax 9", "copies", "products"]


@pytest.mark.parametrize("config", CONFIGS)
def test_prompt_ring_holds_whichever_warp_is_late(config):
    for n in (1, 2, 3, 4, 6, 9):
        for seed in range(2):
            prompt_run(config, n, seed=seed)
        for late in [(w,) for w in WARPS] + [("watcher 2", "watcher 3")]:
            prompt_run(config, n, seed=7, late=late)
    for n in (2, 6):
        for warp in WARPS[:6]:
            for turns in range(0, 14):
                prompt_run(config, n, seed=turns, held=(warp, turns))


@pytest.mark.parametrize("config", CONFIGS)
def test_prompt_block_ends_clean_when_a_wait_runs_out(config):
    """Whatever wait runs out: no barrier gets an arrival that its phase does not expect beside bytes in flight, and the block does not end
    before its copies and products."""
    for n in (1, 3, 6):
        for seed in range(60):
            prompt_run(config, n, seed=seed, give_up=0.002 * (1 + seed % 5), late=((), ("watcher 2",), ("copies",), ("products",))[seed % 4])


# ---- decode: copies, eight compute warps in two teams, two finishing warps ----


def decode_run(slots, pieces, **schedule):
    """A CTA over pieces of so many tiles each."""
    source = _source("attn_decode.cu")
    careful = all(_only_if_ok(source, f"mbar_arrive(&hd->{b}[") for b in ("q_empty", "empty", "part_full", "part_empty"))
    drained = "issued" in source
    run = Run(**schedule)
    full, empty = [Bar(1) for _ in range(slots)], [Bar(4) for _ in range(slots)]
    q_full, q_empty = [Bar(1), Bar(1)], [Bar(8), Bar(8)]
    part_full, part_empty = [Bar(8), Bar(8)], [Bar(2), Bar(2)]
    content, queries, parts = [None] * slots, [None, None], [[None] * 8, [None] * 8]

    def copy(bar, where, i, what):
        where[i] = None
        bar.arrive(tx=1)
        run.copies.append((bar, lambda: where.__setitem__(i, what)))

    def copies():
        issued = q_issued = 0
        ok = True
        for number, tiles in enumerate(pieces):
            b = number & 1
            ok = yield q_empty[b], ((number >> 1) & 1) ^ 1
            if not ok:
                break
            copy(q_full[b], queries, b, number)
            q_issued += 1
            for _ in range(tiles):
                s = issued % slots
                ok = yield empty[s], ((issued // slots) & 1) ^ 1
                if not ok:
                    break
                copy(full[s], content, s, issued)
                issued += 1
            if not ok:
                break
        if drained:
            for at in range(max(0, issued - slots), issued):
                yield full[at % slots], (at // slots) & 1, True
            for at in range(max(0, q_issued - 2), q_issued):
                yield q_full[at & 1], (at >> 1) & 1, True

    def compute(warp):
        ok, count = True, 0
        for number, tiles in enumerate(pieces):
            b = number & 1
            ok = ok and (yield q_full[b], (number >> 1) & 1)
            run.check(queries[b] == number, "queries", queries[b], "for", number)
            if ok or not careful:
                q_empty[b].arrive()
            for _ in range(tiles):
                if count & 1 == warp >> 2:
                    s = count % slots
                    ok = ok and (yield full[s], (count // slots) & 1)
                    run.check(content[s] == count, "a tile", content[s], "for", count)
                    yield None
                    run.check(content[s] == count, "a tile in use is overwritten")
                    if ok or not careful:
                        empty[s].arrive()
                count += 1
            ok = ok and (yield part_empty[b], ((number >> 1) & 1) ^ 1)
            parts[b][warp] = number
            if ok or not careful:
                part_full[b].arrive()

    def finish():
        ok = True
        for number in range(len(pieces)):
            b = number & 1
            ok = ok and (yield part_full[b], (number >> 1) & 1)
            run.check(parts[b] == [number] * 8, "parts", parts[b], "for", number)
            yield None
            run.check(parts[b] == [number] * 8, "parts in use are overwritten")
            if ok or not careful:
                part_empty[b].arrive()

    run.warps = {"copies of tiles": copies(), "finish 0": finish(), "finish 1": finish(), **{f"compute {w}": compute(w) for w in range(8)}}
    run.go()


PIECES = [[1], [2, 1], [9], [3, 1, 1, 4, 2], [1] * 9, [12, 5]]


@pytest.mark.parametrize("slots", [4, 8])
def test_decode_ring_holds_whichever_warp_is_late(slots):
    for pieces in PIECES:
        for late in [()] + [(w,) for w in ("copies of tiles", "finish 0", "compute 0", "compute 5", "copies")] + [("compute 0", "compute 1", "compute 2", "compute 3")]:
            for seed in range(4):
                decode_run(slots, pieces, seed=seed, late=late)
        for warp in ("copies of tiles", "finish 1", "compute 3", "compute 4"):
            for turns in range(12):
                decode_run(slots, pieces, seed=turns, held=(warp, turns))


@pytest.mark.parametrize("slots", [4, 8])
def test_decode_block_ends_clean_when_a_wait_runs_out(slots):
    for pieces in PIECES:
        for seed in range(150):
            decode_run(slots, pieces, seed=seed, give_up=0.005 * (1 + seed % 5), late=((), ("compute 2",), ("copies",), ("finish 0",))[seed % 4])
