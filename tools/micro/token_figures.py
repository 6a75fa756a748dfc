"""Figures around the token operators that no kernel profile holds: the card's copy and product rates, what autograd costs around two empty calls, and what --act_bits 8 keeps
and costs in the 192 x 640 training step.  python tools/micro/token_figures.py [rates] [host] [step]"""
import os
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)
import torch  # noqa: E402


def rates():
    def seconds(f, n=20):
        for _ in range(5):
            f()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            f()
        b.record()
        torch.cuda.synchronize()
        return a.elapsed_time(b) / n * 1e-3

    for mb in (64, 256, 1024, 4096):
        x = torch.empty(mb << 18, device="cuda")
        y = torch.empty_like(x)
        print("copy of %d MiB: %.2f TB/s" % (mb, 8 * x.numel() / seconds(lambda: y.copy_(x)) / 1e12), flush=True)
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        a, b = (torch.randn(8192, 8192, device="cuda", dtype=dt) for _ in range(2))
        print("8192^3 product, %s: %.0f TFLOP/s" % (dt, 2 * 8192 ** 3 / seconds(lambda: a @ b) / 1e12), flush=True)


def host():
    from movedepth_amd import ops

    x, w, b = (torch.ones(s, device="cuda", requires_grad=True) for s in ((64, 64), (64,), (64,)))
    g = torch.ones(64, 64, device="cuda")

    class Empty(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, b):
            ctx.save_for_backward(x, w, b)
            return torch.empty_like(x)

        @staticmethod
        def backward(ctx, g):
            return tuple(torch.empty_like(t) for t in ctx.saved_tensors)

    def us(f, n=2000):
        for _ in range(200):
            torch.autograd.grad(f(), (x, w, b), g)
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(n):
            torch.autograd.grad(f(), (x, w, b), g)
        torch.cuda.synchronize()
        return (time.perf_counter() - t) / n * 1e6

    for _ in range(3):
        print("64 x 64, forward and backward: a function without kernels %.0f us, torch's layer norm %.0f us, ops.layer_norm %.0f us"
              % (us(lambda: Empty.apply(x, w, b)), us(lambda: torch.nn.functional.layer_norm(x, (64,), w, b)), us(lambda: ops.layer_norm(x, w, b))), flush=True)


def step():
    import numpy as np

    from movedepth_amd import miopen_setup
    from movedepth_amd.options import MovedepthOptions
    from movedepth_amd.synthetic import make_inputs
    from movedepth_amd.trainer import Trainer

    miopen_setup.use_shipped_cache(0)
    find = ["--miopen_find", "2" if miopen_setup.find_db_hits(0) else "1"]
    for extra in ([], ["--act_bits", "8"], ["--match_attention", "2"], ["--match_attention", "2", "--act_bits", "8"]):
        opt = MovedepthOptions().parse(["--height", "192", "--width", "640", "--num_depth_bins", "96", "--batch_size", "6", "--convex_up", "--weights_init", "scratch"]
                                       + find + extra)
        torch.manual_seed(0)
        np.random.seed(0)
        t = Trainer(opt)
        t.set_train()
        inputs = make_inputs(6, 192, 640, opt.frame_ids, seed=1, device=t.device)
        for _ in range(3):
            t.train_step(dict(inputs))
        torch.cuda.synchronize()
        at = time.perf_counter()
        for _ in range(10):
            t.train_step(dict(inputs))
        torch.cuda.synchronize()
        ms = (time.perf_counter() - at) * 100
        t.model_optimizer.zero_grad(set_to_none=True)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out, losses = t.process_batch(dict(inputs), is_train=True)
        torch.cuda.synchronize()
        kept = torch.cuda.memory_allocated() - before
        losses["loss"].backward()
        print("192 x 640, batch 6 %s: %.2f ms a step, %.2f GB kept between the passes" % (" ".join(extra) or "(default)", ms, kept / 1e9), flush=True)
        del t, out, losses, inputs
        torch.cuda.empty_cache()


if __name__ == "__main__":
    for name in sys.argv[1:] or ("rates", "host", "step"):
        {"rates": rates, "host": host, "step": step}[name]()
