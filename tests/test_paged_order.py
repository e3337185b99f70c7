"""What the many-row form of the paged attention promises about the order of its products, read from its source: a product that may
overwrite an operand of another one cannot be caught by running it."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sharpmind_b200", "csrc", "smc_paged_prompt.cu")


def test_scores_wait_for_the_product_whose_weights_they_overwrite():
    """The scores of step x go to the columns that hold the weights of step x - 2, and no rule orders two products of different accumulators: between the product of
    step x - 2 and those scores the issuing thread waits for the barrier that the product completes, by the parity of that step."""
    text = open(SOURCE).read()
    body = text[text.index("issue_mmas(uint32_t sbase"):text.index("struct PairWalk")]
    events = re.findall(r"mma_ts<|mma_ss<|smc_tc_commit\(bar\(PV_DONE|wait\(PV_DONE \+ TILE_NO, \(uint32_t\)\(x - 2\)\)|smc_tc_fence_after\(\)", body)
    product, scores = events.index("mma_ts<"), events.index("mma_ss<")
    assert product < scores
    assert [e.split("(")[0] for e in events[product + 1:scores]] == ["smc_tc_commit", "wait", "smc_tc_fence_after"]
