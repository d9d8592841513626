"""Python threads beside the W8A8 operators: while a call waits for room in the device's launch queue, the others run."""
import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls():
    from lightcompress_b200 import block_ops as bo, int8_linear as il
    x, one = torch.randn(4, 64, device='cuda'), torch.ones(64, device='cuda')
    w, ws = torch.ones(8, 64, dtype=torch.int8, device='cuda'), torch.ones(8, device='cuda')
    codes, scales = il.act_quant(x)
    q, pos, freq = torch.randn(1, 2, 3, 8, device='cuda'), torch.arange(3, device='cuda'), torch.ones(4, device='cuda')
    return {'act_quant': lambda: il.act_quant(x), 'gated_act_quant': lambda: il.gated_act_quant(x, x),
            'int8_gemm': lambda: il.int8_gemm(codes, scales, w, ws), 'int8_linear': lambda: il.int8_dynamic_forward_func(x, w, ws),
            'residual_norm': lambda: bo.residual_norm(x, x, weight=one), 'rotary_embed': lambda: bo.rotary_embed(q, None, pos, freq)}


@pytest.mark.parametrize('name', ['act_quant', 'gated_act_quant', 'int8_gemm', 'int8_linear', 'residual_norm', 'rotary_embed'])
def test_other_threads_run_while_a_launch_waits(name):
    """The device is busy for about a second, the queue takes about a thousand launches, so the loop below waits for most of that
    second.  A thread that wakes every millisecond may not stand still for a quarter of it."""
    call = _calls()[name]
    call()
    torch.cuda.synchronize()
    seen, done = [], threading.Event()

    def tick():
        while not done.is_set():
            seen.append(time.perf_counter())
            time.sleep(0.001)
    thread = threading.Thread(target=tick)
    thread.start()
    time.sleep(0.05)
    torch.cuda._sleep(1_900_000_000)                       # clocks: ends by itself
    begin = time.perf_counter()
    for _ in range(3000):
        call()
    took = time.perf_counter() - begin
    done.set()
    thread.join()
    torch.cuda.synchronize()
    longest = max(b - a for a, b in zip(seen, seen[1:]))
    print(f'{name}: the calls took {took:.3f} s, the longest gap of the other thread was {longest:.4f} s')
    assert longest < 0.25
