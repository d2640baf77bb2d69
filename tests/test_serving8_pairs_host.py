"""The CTA-pair kernel of the 8-bit linear layer, read from its source: which tile width a shape gets, and that no remote arrive is
left unwaited when a CTA of the pair leaves."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parent.parent / "deplodock_b200" / "csrc" / "emk_gemm_e4m3_sm100.cu").read_text()
SMS = 148

#: shape -> width of the tiles; several tiles a pair, ragged rows and columns, odd numbers of K slices (1040 = 8 * 128 + 16)
PAIR_SHAPES = {
    (4096, 6144, 2048): 256, (3999, 6136, 1040): 256, (5000, 9992, 400): 256,
    (1024, 6144, 2048): 192, (1001, 6136, 1040): 192, (769, 6008, 272): 192,
    (1024, 4736, 1024): 128, (1000, 4728, 1040): 128, (300, 2048, 528): 128,
}


def _python(expression: str) -> str:
    return expression.replace("&&", " and ").replace("||", " or ").replace("/", "//").replace("!", " not ")


def few_rows(M, N, K):
    body = re.search(r"bool few_rows\(.*?\) \{\n(.*?)\n\}", SOURCE, re.S).group(1)
    first, last = re.fullmatch(r"\s*if \((.*?)\) return true;\n\s*return (.*?);", body).groups()
    return any(eval(_python(e), {}, dict(M=M, N=N, K=K, BM=128)) for e in (first, last))


def tile_width(M, N, pairs=SMS // 2):
    weights = {int(w): int(c) for w, c in re.findall(r"cost\((\d+), (\d+)\)", SOURCE)}
    assert set(weights) == {256, 192, 128}
    cost = {w: -(-(-(-M // 256) * -(-N // w)) // pairs) * c for w, c in weights.items()}
    if cost[128] < cost[192] and cost[128] < cost[256]:
        return 128
    return 192 if cost[192] < cost[256] else 256


@pytest.mark.parametrize("shape", PAIR_SHAPES)
def test_each_tile_width_is_reached(shape):
    M, N, K = shape
    assert not few_rows(M, N, K) and tile_width(M, N) == PAIR_SHAPES[shape]


def test_every_remote_arrive_is_waited_for():
    """An epilogue warp tells the leader that it has drained an accumulator; the leader's MMA warp waits for that before it fills
    the accumulator again, two tiles on. An arrive for an accumulator that is not filled again would be waited for by nobody."""
    kernel = SOURCE[SOURCE.index("gemm2_e4m3_kernel(const"):SOURCE.index("// Few rows:")]
    arrives = re.findall(r"if \((.*?)\) mbar_arrive_cluster_relaxed\(mapa_u32\(smem_u32\(&bars->tmem_empty\[acc\]\), 0\)\);", kernel)
    assert len(arrives) == kernel.count("mbar_arrive_cluster") == 1
    guard = _python(re.sub(r"^lane == 0( && )?", "", arrives[0]) or "1")
    for npairs in (1, 2, 3, 74):
        for ntiles in (1, 2, 3, 73, 74, 75, 147, 148, 149, 221, 222, 223, 400):
            for pair in {0, 1, npairs - 1} & set(range(min(npairs, ntiles))):
                tiles = range(pair, ntiles, npairs)
                sent = [0, 0]
                for local, tile in enumerate(tiles):
                    sent[local & 1] += bool(eval(guard, {}, dict(tile=tile, npairs=npairs, ntiles=ntiles)))
                # the MMA warp's first wait of an accumulator finds it free; each later one takes one phase of arrives
                waited = [max(0, len(range(acc, len(tiles), 2)) - 1) for acc in (0, 1)]
                assert sent == waited, (npairs, ntiles, pair)


def test_the_ring_is_drained_before_a_cta_leaves():
    """The leader's MMA warp releases the peer's stages by remote commits; the peer's producer waits for the last ones."""
    kernel = SOURCE[SOURCE.index("gemm2_e4m3_kernel(const"):SOURCE.index("// Few rows:")]
    producer = kernel[kernel.index("if (warp == P8_TMA_WARP) {"):kernel.index("} else if (warp == P8_MMA_WARP)")]
    tail = producer[producer.rindex("for (int i = 0; i < P8_STAGES"):]
    assert "mbar_wait(&bars->empty[stage], phase ^ 1u" in tail
    for stages in (3,):
        for fills in range(0, 12):  # phases as the barrier has them: every fill is released once
            released = [len(range(s, fills, stages)) for s in range(stages)]
            stage, phase = fills % stages, (fills // stages) & 1
            for _ in range(stages):
                # waiting for parity phase ^ 1 returns once as many releases as fills of this stage have arrived
                assert released[stage] == 0 or (released[stage] - 1) & 1 == phase ^ 1
                stage += 1
                if stage == stages:
                    stage, phase = 0, phase ^ 1
