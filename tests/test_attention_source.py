"""What the order of the attention tiles' steps rests on, read in their source."""
import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parents[1] / "ptq_int8_lab_b200" / "csrc" / "ptq8_attention_tc.cuh"


def test_waits_for_tmem_loads_name_their_registers():
    """A load's registers hold nothing before the wait; only one that names them keeps the compiler from using them before it."""
    text = SOURCE.read_text()
    loads = re.findall(r"^ +(?:if \(.*\) )?tmem_(?:load8|ld16)\(.*, ([a-z\[\] &()+0-9]+)\);", text, re.M)
    waits = re.findall(r"^ +tmem_wait_ld\((.*?)\);", text, re.M)
    assert len(loads) >= 6 and len(waits) >= 6
    assert all(w.strip() for w in waits), waits
    assert {v.split("[")[0] for v in loads} <= {w.split("[")[0] for w in waits} | {"coming"}


def test_parameters_are_announced_before_the_keys_that_scores_follow():
    """A half that skipped items may be phases early at the parameters' barrier: it relies on the scores, and those on this order."""
    text = SOURCE.read_text()
    assert 0 < text.index("mbar_arrive(par_full") < text.index("mbar_arrive(k_full")
    assert text.index("wait(par_full") < text.index("wait(s_full")
    assert text.count("mbar_arrive(par_full") == text.count("mbar_arrive(k_full") == 1
