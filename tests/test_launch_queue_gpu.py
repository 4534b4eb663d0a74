"""Calls that wait for room in the launch queue leave Python's lock to other threads."""
import threading
import time

import pytest
import torch

import flash_attn_with_score_b200 as F

pytestmark = pytest.mark.gpu


def _calls():
    cache = F.KVCache4(4, 16, 2, 64)
    table = torch.arange(2, dtype=torch.int32, device="cuda").view(1, 2)
    lengths = torch.full((1,), 20, dtype=torch.int32, device="cuda")
    x = torch.randn((1, 2, 1, 64), device="cuda").half()
    kv = torch.randn((1, 2, 40, 64), device="cuda").half()
    return {"write": lambda: F.kv_cache_write(cache, x, x, table, lengths), "read": lambda: F.kv_cache_read(cache, table, lengths, 3),
            "attention": lambda: F.attention_with_kv_cache(x, cache, table, lengths),
            "window": lambda: F.attention_with_window(x, kv, kv, 10, 1)}


@pytest.mark.parametrize("name", ["write", "read", "attention", "window"])
def test_other_threads_run_while_the_queue_is_full(name):
    call = _calls()[name]
    for _ in range(3):
        call()
    torch.cuda.synchronize()
    gaps, stop, going = [], threading.Event(), threading.Event()

    def tick():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            gaps.append(now - last)
            last = now
            going.set()

    other = threading.Thread(target=tick)
    other.start()
    going.wait()
    try:
        t0 = time.perf_counter()
        torch.cuda._sleep(int(0.5 * 1.8e9))  # half a second or so, behind which the queue fills
        for _ in range(4000):
            call()
        took = time.perf_counter() - t0
    finally:
        stop.set()
        other.join()
    torch.cuda.synchronize()
    assert took > 0.3, "the calls waited for the queue"
    assert max(gaps) < 0.5 * took, f"another thread stood still for {max(gaps):.2f} s of {took:.2f}"
    assert F.device_status() == 0
