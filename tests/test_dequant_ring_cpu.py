"""Stages of the dequant GEMM's ring: each belongs to the same converter groups every time it is filled."""
import re

from sneppx_alg_b200 import _build


def test_a_stage_belongs_to_the_same_groups_each_time():
    """K-block i is in stage i // KPS modulo the ring and is taken by group i modulo NG: the same group for every turn of the ring needs a ring of whole
    turns of the groups."""
    text = (_build.CSRC / "gemm_dq.cu").read_text()
    most = int(re.search(r"DQ_MAX_STAGES = (\d+)", text).group(1))
    for bt in (16, 32, 64, 128):
        groups, budget = (4 if bt == 64 else 2), (98304 if bt <= 32 else 196608)
        assert "NG = BT == 64 ? 4 : 2" in text and "BUDGET = CTAS == 2 ? 98304 : 196608" in text and "p.stages = ROOM / TURN * TURN;" in text
        for kps in (1, 2):
            room, turn = min(budget // (16384 + kps * bt * 256), most), max(groups // kps, 1)
            stages = room // turn * turn
            assert stages >= 2
            owner = {}
            for i in range(8 * stages * kps):
                assert owner.setdefault((i // kps % stages, i % kps), i % groups) == i % groups, (bt, kps, i)
