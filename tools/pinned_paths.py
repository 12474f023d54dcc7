#!/usr/bin/env python3
"""ClownResampler_LowLevel_ResampleBulk from HOST memory, pageable against page-locked buffers, by the way cr_run_host treats
page-locked ones (CLOWNRESAMPLER_AMD_HOST_DIRECT, read once per process: every leg is a child process):
    0  staged like pageable memory (hipMemcpyAsync up, kernel, hipMemcpyAsync down; the round-3 behaviour)
    1  the kernel reads the caller's input in place, the output is staged
    2  ONE launch reads the input and writes the output in place (nothing staged)
   -1  the library's rule
Workloads: cfg 2 (10 min stereo) and shorter / wider ones.  pinned (6.1 ms) lost to pageable (4.8 ms)."""
import json
import os
import subprocess
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CASES = [("cfg2", 3, 2, (44100, 48000, 44100), 26460000), ("1min", 3, 2, (44100, 48000, 44100), 2646000), ("cfg4", 3, 8, (48000, 44100, 44100), 28800000),
         ("cfg3", 8, 2, (8000, 96000, 8000), 4800000), ("dn8", 3, 2, (44100, 8000, 8000), 26460000)]


def child(mode):
    sys.path.insert(0, ROOT)
    sys.path.insert(0, os.path.join(ROOT, "tests"))
    import numpy as np
    import torch
    torch.cuda.init()
    import clownresampler_amd as cr
    res = {}
    for name, radius, ch, rates, frames in CASES:
        api = cr.load(radius)
        pre = api.precomputed()
        fresh = api.LowLevel_State()
        assert api.LowLevel_Init(fresh, ch, *rates)
        R = fresh.lowest_level.integer_stretched_kernel_radius
        n_out = int(api.CountOutputFrames(fresh, frames))
        rng = np.random.default_rng(1)
        pcm = np.zeros((frames + 2 * R) * ch, dtype=np.int16)
        pcm[R * ch:(R + frames) * ch] = rng.integers(-32768, 32768, size=frames * ch, dtype=np.int16)
        out = np.zeros((n_out + 1) * ch, dtype=np.int32)

        def once(src, dst):
            st = cr.LowLevel_State.from_buffer_copy(fresh)
            t0 = time.perf_counter()
            got, left, ran_out = api.LowLevel_ResampleBulk(st, pre, src, frames, n_out + 1, output=dst)
            dt = (time.perf_counter() - t0) * 1e3
            assert got.size == n_out * ch and left == 0 and ran_out == 1
            return dt

        pageable = [once(pcm, out) for _ in range(5)]
        pin_in = torch.empty(pcm.size, dtype=torch.int16).pin_memory()
        pin_out = torch.zeros(out.size, dtype=torch.int32).pin_memory()
        pin_in.numpy()[:] = pcm
        pinned = [once(pin_in.numpy(), pin_out.numpy()) for _ in range(5)]
        same = bool(np.array_equal(pin_out.numpy()[: n_out * ch], out[: n_out * ch]))
        res[name] = {"pageable_ms": min(pageable[1:]), "pinned_ms": min(pinned[1:]), "pinned_first_ms": pinned[0], "same": same,
                     "MB": (pcm.nbytes + n_out * ch * 4) / 1e6}
        del pin_in, pin_out
    print(json.dumps(res))


def main():
    if len(sys.argv) > 1 and sys.argv[1] == "child":
        return child(sys.argv[2])
    print("%-6s %8s | %s" % ("case", "MB", "  ".join("mode %2s: pageable / pinned ms" % m for m in ("0", "1", "2", "-1"))))
    rows = {}
    for mode in ("0", "1", "2", "-1"):
        env = dict(os.environ)
        if mode == "-1":
            env.pop("CLOWNRESAMPLER_AMD_HOST_DIRECT", None)
        else:
            env["CLOWNRESAMPLER_AMD_HOST_DIRECT"] = mode
        r = subprocess.run([sys.executable, os.path.abspath(__file__), "child", mode], env=env, capture_output=True, text=True, timeout=900)
        if r.returncode != 0:
            print("mode %s failed: %s" % (mode, r.stderr[-800:]))
            continue
        rows[mode] = json.loads(r.stdout.strip().splitlines()[-1])
    for name, *_ in CASES:
        cells = []
        for mode in ("0", "1", "2", "-1"):
            c = rows.get(mode, {}).get(name)
            cells.append("%26s" % ("%.2f / %.2f%s" % (c["pageable_ms"], c["pinned_ms"], "" if c["same"] else " DIFFERENT") if c else "-"))
        print("%-6s %8.1f | %s" % (name, rows[next(iter(rows))][name]["MB"], "  ".join(cells)))


if __name__ == "__main__":
    main()
