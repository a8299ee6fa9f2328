"""Forms of the norm's backward (CPU): those that the library holds are those that some row length and type is launched with."""

import re

from dist_moe_b200 import build

TEXT = (build.CSRC / "add_rmsnorm.cu").read_text()


def _chosen():
    """The rule of the host side, walked over every row length of the register forms: (fp32 stream, row to a warp, pieces, stages)."""
    found = set()
    for wide in (1, 2):
        for vec in range(1, 2049):
            warp, pieces = (True, 4) if vec * 8 <= 1024 else (False, 2 if vec <= 1024 else 4)
            threads = 128 if warp else -(-vec // (32 * pieces)) * 32
            two = 220 * 1024 // (2 * threads * pieces * (1 + 2 * wide) * 16 + 2048)
            found.add((wide == 2, warp, pieces, 2 if two >= 1 else 1))
    return found


def test_every_form_of_the_backward_is_launched_by_some_size():
    build.build()
    log = (build.LIB_DIR / "ptxas.log").read_text()
    held = {(m[1] == "f", m[2] == "1", int(m[3]), int(m[4]))
            for m in re.finditer(r"add_rmsnorm_bwd_kernelI(f|13__nv_bfloat16)Lb([01])ELi(\d)ELi(\d)E", log)}
    assert held == _chosen()


def test_the_rule_that_is_walked_over_is_the_sources():
    for piece in ("if (D <= 1024) return run(std::true_type{}, integral_constant<int, 4>{}, 128);", "kPieces = kVec * (1 + 2 * kWide)",
                  "if (vec <= 2 * kNormThreads) return run(std::false_type{}, integral_constant<int, 2>{}", "220 * 1024 / (stages * stage_bytes(threads) + 2048)"):
        assert piece in TEXT, piece
