"""Kernels that issue bulk copies end, or use the places of the copies for something else, only behind a wait for each that was issued, where a wait ran
out of its limit too: read from the sources, since no run shows it."""

import re

import pytest

from test_device_sources_cpu import source


def ring(limits_at, issued, stages):
    """The loops of the kernel for few rows, written out: the wait number `limits_at` runs out.  Returns what was waited for, (stage, phase) of each copy."""
    waited, stage, phase, done, total = [], 0, 0, 0, issued

    def next_stage(stage, phase):
        return (0, phase ^ 1) if stage + 1 == stages else (stage + 1, phase)

    on_way = min(stages, total)
    while done < on_way:
        waited.append((stage, phase))
        if done == limits_at:
            break
        on_way = min(on_way + 1, total)
        stage, phase = next_stage(stage, phase)
        done += 1
    while done < on_way:
        waited.append((stage, phase))
        stage, phase = next_stage(stage, phase)
        done += 1
    return waited, on_way


@pytest.mark.parametrize("stages", [4, 6])
@pytest.mark.parametrize("issued", [0, 1, 3, 4, 5, 23])
def test_every_copy_that_was_issued_is_waited_for(stages, issued):
    for limits_at in range(issued + 1):
        waited, on_way = ring(limits_at, issued, stages)
        assert set(waited) >= {(n % stages, n // stages & 1) for n in range(max(0, on_way - stages), on_way)}
        assert waited[-1:] == ([((on_way - 1) % stages, (on_way - 1) // stages & 1)] if on_way else [])


def test_the_kernel_for_few_rows_over_4_bit_pages_waits_for_what_it_issued():
    """`done` counts the waits that were held, the second loop begins where the first one ended, and nothing else lies between it and the first use of the ring for the sums."""
    text = source("vx_prefix_fp4.cu")
    text = text[text.index("prefix_rows_fp4_kernel("):]
    text = text[:re.search(r"\n}\n", text).end()]
    first, second = [m.start() for m in re.finditer(r"for \(; done < issued; \+\+done\) {", text)]
    body = text[second:text.index("\n  }\n", second)]
    assert "break" in text[first:second] and "break" not in body and "return" not in text[first:]
    assert re.search(r"mbar_wait\(&full_s\[warp\]\[stage\], phase, p\.status", body) and "next_stage();" in body
    assert not re.search(r"\b(done|stage|phase) ?=(?!=)", text[first:second + len(body)].replace("for (; done", ""))
    assert text[second + len(body):].lstrip("\n }").startswith("named_bar_sync(")
    assert text.index("bulk_load(") < first and "bulk_load(" not in text[second:]


def walked_back(slots, calls, fetched):
    """The end of the warp that fetches units for the tiles: the slots and phases that it waits for."""
    slot, phase = 0, 0
    armed = []
    for _ in range(calls):
        armed.append((slot, phase))
        slot += 1
        if slot == slots:
            slot, phase = 0, phase ^ 1
    waits = []
    i = 0
    while i < slots and i <= fetched:
        if slot == 0:
            phase ^= 1
        slot = (slots if slot == 0 else slot) - 1
        waits.append((slot, phase))
        i += 1
    return armed, waits


@pytest.mark.parametrize("slots", [1, 2, 3, 6])
@pytest.mark.parametrize("fetched", range(9))
def test_the_last_units_of_the_tiles_are_waited_for(slots, fetched):
    """Ended as it should (a slot for the end behind those of the tiles), or given up with or without a slot asked for in vain."""
    for calls in (fetched, fetched + 1):
        armed, waits = walked_back(slots, calls, fetched)
        assert set(armed[-slots:]) <= set(waits)


def test_the_warp_that_fetches_for_the_tiles_waits_whether_it_gave_up_or_not():
    """It can have issued all of its copies before a loader's wait runs out."""
    text = source("vx_prefix_tiles.cu")
    text = text[text.index("next_raw(e, kRawEnd, 0)"):]
    text = text[:text.index("cp_async_wait_all()")]
    assert re.search(r"for \(int e = 0; e < 2; \+\+e\)\s*for \(int i = 0; i < \(e \? Shape::kRawV : Shape::kRawK\) && i <= fetched; \+\+i\) {", text)
    assert "mbar_wait(&bar.raw[stream][e].full[raw_slot[e]], raw_phase[e], p.status" in text and "if (!ok)" not in text
