"""The prompt's kernel of the attention over a shared prompt: a wait on a barrier of a ring knows the phase by its parity, so nobody may let
the barrier go on by two phases before the wait has been passed.  Read from the source: a missing wait need not show in any run."""

import re
from pathlib import Path

KERNEL = Path(__file__).resolve().parents[1] / "csrc" / "shared_prefix_tcgen05.cu"


def test_the_first_key_is_seen_before_its_stage_is_filled_again():
    """The producer of V waits for the first K without consuming it: a K stage is freed by the scores alone, which do not need V."""
    text = re.sub(r"//[^\n]*", "", KERNEL.read_text())
    keys, values = text.index("map_k, k_full(turn.st)"), text.index("map_v, v_full(turn.st)")
    first = text.index("mbar_wait(k_full(0), 0", keys)
    seen = re.search(r"mbar_arrive\((\w+)\)", text[first:values])
    assert seen, "V's producer does not say that it has seen the first K"
    barrier = seen.group(1)
    # one arrival, one wait, both of the only phase there is; the wait comes before the copy into a stage that was full once
    assert re.search(rf"mbar_init\({barrier}, 1\)", text) and text.count(f"mbar_arrive({barrier})") == 1
    producer = text[text.index("if (warp == 0) {\n", text.index("regs_give<REGS_ISSUE>()")) : keys]
    wait = re.search(rf"if \(issued == stages && !mbar_wait\({barrier}, 0,", producer)
    assert wait, "the producer of K fills a stage again without it"
    assert producer.index("mbar_expect_tx(k_full") > wait.start()
