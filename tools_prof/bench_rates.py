"""The card's rates that the operators' floors are counted at: a large copy and large bf16 products of the library."""
import time
import torch


def seconds(f, n=20):
    for _ in range(5):
        f()
    torch.cuda.synchronize(); t0 = time.perf_counter()
    for _ in range(n):
        f()
    torch.cuda.synchronize()
    return (time.perf_counter() - t0) / n


x = torch.randn(1 << 30, device="cuda", dtype=torch.bfloat16)
y = torch.empty_like(x)
print(f"copy of 2 GiB: {4 * x.numel() / seconds(lambda: y.copy_(x)) / 1e12:.2f} TB/s read and written", flush=True)
for M, N, K in ((8192, 8192, 8192), (4096, 65536, 2048)):
    a, b = (torch.randn(r, K, device="cuda").bfloat16() for r in (M, N))
    bt = b.t().contiguous()
    for what, f in (("second operand's rows along K", lambda: a @ b.t()), ("along N", lambda: a @ bt)):
        print(f"product {M} x {N} x {K}, {what}: {2 * M * N * K / seconds(f) / 1e12:.0f} TFLOP/s", flush=True)
