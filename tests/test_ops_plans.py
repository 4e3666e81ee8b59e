"""How calls with changed scores are cut (no GPU here)."""
from gqa_kernels.dispatch import scored_plan
from gqa_kernels.paged import SCORED_THREE_FILL, scored_paged_plan


def test_three_chunks_for_two_only_where_they_are_faster_for_equal_and_unequal_lengths():
    """Of a batch over pages whose lengths the host does not know."""
    seen = set()
    for D in (64, 128):
        for B in (1, 2, 3, 4, 8, 12):
            for Hkv in (1, 2, 4, 8):
                for G in (1, 4, 8):
                    for Sq in (64, 150, 256, 500, 1100):
                        for ml in (1200, 2600, 5000, 9000, 16000):
                            args = (B, G * Hkv, Hkv, Sq, ml, 256, True, D)
                            if G * Sq <= 128:
                                continue
                            p, (route, chunks) = scored_plan(*args), scored_paged_plan(*args)
                            assert route == p.kind
                            if p.kind != "chunks":
                                assert chunks == 0
                                continue
                            three = B > 1 and p.splits == 2 and (D == 64 or p.workgroups / 512 <= SCORED_THREE_FILL)
                            assert chunks == (3 if three else p.splits), args
                            seen.add((D, p.splits == 2, three))
    assert {(64, True, True), (128, True, True), (128, True, False), (128, False, False)} <= seen
    # 4 x 256 and 8 x 256 tokens of 32 / 8 heads: two chunks fill the slots of one round, three would take a second.
    assert scored_paged_plan(4, 32, 8, 256, 9000, 256, True, 128) == ("chunks", 2)
    assert scored_paged_plan(8, 16, 8, 256, 7659, 256, True, 128) == ("chunks", 2)
