"""Barriers of the dequant GEMM's ring: each belongs to the same converter groups every time it is armed."""
import re

from sneppx_alg_b200 import _build


def test_a_barrier_belongs_to_the_same_groups_each_time():
    """K-block i is in stage i // KPS modulo the ring, is told by the barrier of that stage for even or odd turns, and is taken by group i modulo NG."""
    text = (_build.CSRC / "gemm_dq.cu").read_text()
    most = int(re.search(r"DQ_MAX_STAGES = (\d+)", text).group(1))
    assert "NG = BT == 64 ? 4 : 2" in text and "BUDGET = CTAS == 2 ? 98304 : 196608" in text
    # producer, MMA warps and converters name it alike
    assert "full[(i / p.stages & 1) * DQ_MAX_STAGES + s]" in text and text.count("full[(turn & 1) * DQ_MAX_STAGES + s], turn >> 1 & 1") == 2
    alone = True
    for bt in (16, 32, 64, 128):
        groups, budget = (4 if bt == 64 else 2), (98304 if bt <= 32 else 196608)
        for kps in (1, 2):
            stages = min(budget // (16384 + kps * bt * 256), most)
            assert stages >= 2
            owner, single = {}, {}
            for i in range(8 * stages * kps):
                st, g = i // kps, i % groups
                assert owner.setdefault((st % stages, st // stages % 2, i % kps), g) == g, (bt, kps, i)
                alone &= single.setdefault((st % stages, i % kps), g) == g
    assert not alone          # one barrier a stage would not do
