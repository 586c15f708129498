"""The host model of the span tile kernel's pipeline (test_span_tile_protocol) against
the kernel's source: the barriers' counts, each warp's waits and arrivals in their
order and with their parities are read off the source and compared with the model's.
The model also gets the V rows that a softmax warp zeroes in the ring, and fails in
some of its random orders for every wait that is left out."""
import random
import re

import pytest

from test_span_tile_protocol import SOURCE, STAGES, Tile

KERNEL = re.sub(r"//[^\n]*", "", SOURCE[SOURCE.index("span_tiles_kernel(const SpanParams"):
                                        SOURCE.index("cudaError_t launch_tiles(")])
NAMES = {"q_full": "q_full", "o_full": "o_full", "kBarSFull": "s_full", "kBarSRead": "s_read",
         "kBarPFull": "p_full", "kBarPvDone": "pv_done", "kBarKvFull": "kv_full", "kBarKvEmpty": "kv_empty",
         "kBarDrain": "drain"}


def section(start, end):
    return KERNEL[KERNEL.index(start):KERNEL.index(end)]


PRODUCERS = section("if (warp == 0 || warp == 3)", "if (warp <= 2)")
S_ISSUER = section("const uint64_t q_desc", "const uint64_t v_desc")
PV_ISSUER = section("const uint64_t v_desc", "umma_commit(bar(kBarDrain")
SOFTMAX = section("setmaxnreg.inc", "named_barrier_sync(2")


def used(text, call):
    """Barriers that `call` names in a piece of the source, in order, as the model calls them."""
    out = []
    for m in re.finditer(rf"\b{call}\(", text):
        arg = text[m.end():m.end() + 60]
        name = re.match(r"(?:bar\()?(q_full|o_full|full|kBar\w+)", arg)
        if name:
            out.append(NAMES.get(name.group(1), name.group(1)))
    return out


def test_the_barriers_counts_are_the_models():
    counts = {NAMES[name]: count for name, count in
              re.findall(r"mbar_init\((?:bar\()?(q_full|o_full|kBar\w+)[^,]*, (\w+)\)", KERNEL)}
    counts.pop("drain")
    quarters = 3
    model = Tile(9, quarters)
    assert set(counts) == set(NAMES.values()) - {"drain"}
    for name, count in counts.items():
        barrier = getattr(model, name)
        barrier = barrier[0] if isinstance(barrier, list) else barrier
        assert barrier.count == (quarters if count == "quarters" else int(count)), name


def test_the_waits_and_arrivals_are_the_models():
    assert used(PRODUCERS, "mbar_wait_sleeping") == ["kv_empty"]
    assert "if (c >= kStages &&" in PRODUCERS and "int issued = 0, stage = 0, parity = 1;" in PRODUCERS
    assert re.search(r"const uint32_t full = bar\(kBarKvFull \+ stage\);", PRODUCERS)
    assert used(PRODUCERS, "mbar_arrive_expect_tx") == ["full"]

    assert used(S_ISSUER, "wait") == ["q_full", "kv_full", "s_read"]
    assert "if (c > 0 && !wait(bar(kBarSRead + ((c - 1) & 1)), ((c - 1) >> 1) & 1)) break;" in S_ISSUER
    assert "wait(bar(kBarKvFull + stage), parity)" in S_ISSUER and "int parity = 0;" in S_ISSUER
    assert used(S_ISSUER, "umma_commit") == ["s_full"]

    assert used(PV_ISSUER, "wait") == ["p_full"]
    assert "wait(bar(kBarPFull + side), (c >> 1) & 1)" in PV_ISSUER
    assert used(PV_ISSUER, "umma_commit") == ["pv_done", "kv_empty", "o_full"]

    assert used(SOFTMAX, "warp_wait") == ["s_full", "pv_done", "o_full"]
    assert used(SOFTMAX, "mbar_arrive") == ["q_full", "s_read", "p_full"]
    assert "warp_wait(bar(kBarSFull + side), parity)" in SOFTMAX and "uint32_t parity = 0;" in SOFTMAX
    assert re.search(r"if \(c >= 2\) \{\s*ok = warp_wait\(bar\(kBarPvDone \+ side\), parity \^ 1u\);", SOFTMAX)
    # P is in Tensor Memory, and the V rows are zeroed and fenced, before P counts as written
    order = [SOFTMAX.index(x) for x in ("kBarPvDone", "tmem_st16(tmem + kColP", "tmem_wait_st()",
                                        "zero_hidden_v_rows", "fence_proxy_async_smem();\n    }", "kBarPFull")]
    assert order == sorted(order)
    assert "(c % kStages) * kChunkBytes + kKvBytes" in SOFTMAX  # the V of chunk c
    assert "!whole && quarter == 0" in SOFTMAX


class Leaving(Tile):
    """The model without the waits for the barriers named `without`."""
    without = ""

    def _agent(self, agent):
        for ok in agent:
            yield (lambda: True) if self.without and self.without in ok.__code__.co_names else ok

    def producer(self, which):
        return self._agent(super().producer(which))

    def s_issuer(self):
        return self._agent(super().s_issuer())

    def pv_issuer(self):
        return self._agent(super().pv_issuer())

    def softmax(self, side, quarter):
        return self._agent(super().softmax(side, quarter))


@pytest.mark.parametrize("without", ["kv_empty", "kv_full", "s_read", "s_full", "p_full", "pv_done", "o_full"])
def test_the_model_sees_every_wait_that_is_left_out(without):
    model = type("Without", (Leaving,), {"without": without})
    with pytest.raises(AssertionError):
        for seed in range(300):
            model(3 * STAGES, 4).run(random.Random(seed))


def test_the_model_ends_with_all_of_its_waits():
    for seed in range(300):
        Leaving(3 * STAGES, 4).run(random.Random(seed))


class Zeroing(Tile):
    """Quarter 0 of a side zeroes rows of chunk c's V between its exponentials and its arrival at
    p_full, or, `late`, after that."""
    late = False

    def softmax(self, side, quarter):
        plain = 0
        for ok in super().softmax(side, quarter):
            yield ok
            if ok.__code__.co_names or quarter != 0:
                continue
            plain += 1  # per chunk: the scores' loads, the exponentials
            if plain % 2 == 0 and not self.late:
                self.zero(side + plain - 2)
            elif plain % 2 == 1 and plain > 1 and self.late:
                self.zero(side + plain - 3)

    def zero(self, c):
        # landed, and P V of this chunk has neither read it nor run ahead
        assert self.ring[c % STAGES]["V"] == c, f"V of chunk {c} is not there"
        assert c not in self.o[c & 1], f"V of chunk {c} was read before it was zeroed"


@pytest.mark.parametrize("quarters", [1, 2, 4])
@pytest.mark.parametrize("chunks", [1, 2, 5, 2 * STAGES, 3 * STAGES + 1])
def test_rows_are_zeroed_between_their_copy_and_the_product(chunks, quarters):
    for seed in range(60):
        Zeroing(chunks, quarters).run(random.Random(seed))


def test_the_model_sees_rows_zeroed_too_late():
    model = type("Late", (Zeroing,), {"late": True})
    with pytest.raises(AssertionError):
        for seed in range(100):
            model(9, 4).run(random.Random(seed))
