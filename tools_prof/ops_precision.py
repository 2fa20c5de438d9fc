"""Relative errors (2-norm) of the stand-alone operators against their 64-bit values over drawn shapes of perf/operators.py:
``ops_precision.py [seed] [cases] [seconds]``. Prints every case above 3.5e-3 and the largest error of each output."""
import os, random, sys, time
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, _ROOT); sys.path.insert(0, os.path.join(_ROOT, "perf"))
import torch
import operators as O

O.own = True
seed, cases, limit = (int(x) for x in (sys.argv[1:] + ["1", "400", "150"][len(sys.argv) - 1:]))
rng = random.Random(seed)
names = {"rotary": ("q", "k", "dq", "dk"), "attention": ("out", "dq", "dk", "dv", "dlam"), "loss": ("loss", "dhidden", "dweight")}
worst, done, t0 = {}, 0, time.time()
for i in range(cases):
    c = O.draw(rng)
    if O.work(c)["flops"] > 3e11:          # (64 bits would take long)
        continue
    state = O.prepare(c, seed + i)
    for name, got, want in zip(names[c["op"]], O.run(state), O.exact(c, seed + i)):
        got, want = got.detach().double(), torch.as_tensor(want, device="cuda").double().reshape(got.shape)
        norm = float(want.norm())
        err = float((got - want).norm()) / norm if norm else float("inf") if bool((got != 0).any()) else 0.0
        key = f"{c['op']} {c.get('dtype', 'bf16')} {name}"
        worst[key] = max(worst.get(key, (0.0, "")), (err, str(c)))
        if not err < 3.5e-3:
            print(f"{err:.2e} {name} {c}", flush=True)
    done += 1
    if done % 50 == 0:
        print(done, "cases", flush=True)
    if time.time() - t0 > limit:
        break
print(f"seed {seed}: {done} cases")
for key in sorted(worst):
    print(f"{key:24s} {worst[key][0]:.2e}")
