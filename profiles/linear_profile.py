"""The linear layers' benchmark cases and the hash heads, for the clock or for a profiler.

  linear_profile.py time                       microseconds a call, back to back, of the heads beside the plain forward, and of the library's products
  linear_profile.py run [NAME ...]             15 calls of each case of perf/operators.py (or of those whose names contain one of NAME), three sets of inputs in turn
  linear_profile.py heads                      15 calls of pb_embed_heads_device: 512 images, 8 heads of 256 channels, f32 and i8
  linear_profile.py trace CSV                  a kernel trace of those (rocprofv3 --kernel-trace), by kernel and grid: calls, median and least time
  linear_profile.py counters CSV [CSV ...]     counter collections (rocprofv3 --pmc), by kernel: the median of each counter
"""
import collections
import csv
import importlib.util
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def short(name):
    return name.split("(")[0].replace("void pbl::", "").replace("pbl::", "")


def trace(path):
    times = collections.OrderedDict()
    with open(path) as f:
        rows = sorted(csv.DictReader(f), key=lambda r: int(r["Start_Timestamp"]))
    for r in rows:
        if "pbl::" in r["Kernel_Name"] or "k_hash_rows" in r["Kernel_Name"]:
            times.setdefault((short(r["Kernel_Name"]), r["Grid_Size_X"]), []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1000)
    for (name, grid), v in times.items():
        v.sort()
        print("%-58s grid %-9s calls %3d  median %8.2f us  least %8.2f" % (name, grid, len(v), v[len(v) // 2], v[0]))


def counters(paths):
    got, took = collections.OrderedDict(), collections.defaultdict(list)
    for path in paths:
        with open(path) as f:
            for r in csv.DictReader(f):
                if "pbl::" in r["Kernel_Name"]:
                    name = short(r["Kernel_Name"])
                    got.setdefault(name, collections.OrderedDict()).setdefault(r["Counter_Name"], []).append(float(r["Counter_Value"]))
                    took[name].append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1000)
    for name, c in got.items():
        us = sorted(took[name])[len(took[name]) // 2]
        mid = {k: sorted(v)[len(v) // 2] for k, v in c.items()}
        print("%-58s median %8.2f us  " % (name, us) + "  ".join("%s %.4g" % kv for kv in mid.items()))
        if us > 200:  # GRBM_GUI_ACTIVE is a sum over 8 XCDs and counts a little before and behind a dispatch: for long kernels alone
            clocks = mid["GRBM_GUI_ACTIVE"] / 8
            print("    %.2f GHz; matrix units busy %.0f %% of the cycles of 1024 SIMDs" % (clocks / us / 1000, 100 * mid["SQ_VALU_MFMA_BUSY_CYCLES"] / clocks / 1024))


def cases():
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    return m


def run(only):
    import torch

    m = cases()
    for case in m.listed():
        if only and not any(o in case["name"] for o in only):
            continue
        sets = [m.prepare(case, s) for s in range(3)]
        for i in range(15):
            m.run(sets[i % 3])
        torch.cuda.synchronize()
        print(case["name"], flush=True)
        del sets
        torch.cuda.empty_cache()


class Heads:
    def __init__(self, n=512, heads=8, d=256):
        import torch

        from pixelbox_amd import capi, linear, synth
        from pixelbox_amd import weights as W

        self.n, self.heads, self.d = n, heads, d
        self.emb = capi.Embedder(W.synthetic_blob(synth.SEED_WEIGHTS, 128, 128, 256), max_batch=n)
        self.s = torch.cuda.current_stream()
        assert self.s.cuda_stream, "a stream of one's own: 0 stands for the embedder's"
        self.emb.set_option(capi.PB_OPT_EMBED_STREAM, self.s.cuda_stream)
        self.emb.set_option(capi.PB_OPT_EMBED_ASYNC, 1)
        self.img = torch.from_numpy(synth.synthetic_images(synth.SEED_IMAGES, 0, n, 128, 128)).cuda()
        g = torch.Generator().manual_seed(1)
        self.head = torch.randint(0, heads, (n,), generator=g, dtype=torch.int32).cuda()
        self.w, self.b = (torch.randn((heads, d, 1280), generator=g) * 0.05).cuda(), torch.randn((heads, d), generator=g).cuda()
        c, s = linear.quantize_rows(self.w.view(-1, 1280))
        self.codes, self.scale = c.view(heads, d, 1280), s.view(heads, d)
        self.u8, self.f32 = torch.zeros((n, d), dtype=torch.uint8, device="cuda"), torch.zeros((n, d), device="cuda")
        self.features = torch.zeros((n, 1280), device="cuda")

    def plain(self):
        self.emb.embed_device(self.img.data_ptr(), self.n, self.u8.data_ptr(), self.f32.data_ptr())

    def only_features(self):
        self.emb.features_device(self.img.data_ptr(), self.n, self.features.data_ptr())

    def with_heads(self, i8):
        w = self.codes if i8 else self.w
        self.emb.heads_device(self.img.data_ptr(), self.n, 3 if i8 else 0, w.data_ptr(), self.heads, self.d, self.head.data_ptr(), self.scale.data_ptr() if i8 else 0,
                              self.b.data_ptr(), self.u8.data_ptr(), self.f32.data_ptr())


def timed(f, n):
    import torch

    for _ in range(3):
        f()
    v = []
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            f()
        b.record()
        b.synchronize()
        v.append(a.elapsed_time(b) * 1000 / n)
    return sorted(v)[3]


def time_all():
    import torch

    torch.cuda.set_stream(torch.cuda.Stream())
    for n, heads in ((1, 8), (40, 8), (512, 8), (512, 64)):
        h = Heads(n, heads)
        print("%d images, %d heads of 256: plain forward %.1f us, features alone %.1f, f32 heads %.1f, 8-bit heads %.1f" % (
            n, heads, timed(h.plain, 20), timed(h.only_features, 20), timed(lambda: h.with_heads(False), 20), timed(lambda: h.with_heads(True), 20)), flush=True)
        del h
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        x, y = (torch.randn(8192, 8192, device="cuda").to(dt) for _ in range(2))
        us = timed(lambda: torch.matmul(x, y.t()), 10)
        print("library product 8192^3 %s: %.0f us, %.0f TFLOP/s" % (dt, us, 2 * 8192 ** 3 / us * 1e-6), flush=True)
    x, y = (torch.randint(-127, 128, (8192, 8192), device="cuda", dtype=torch.int32).to(torch.int8) for _ in range(2))
    us = timed(lambda: torch._int_mm(x, y.t()), 10)
    print("library product 8192^3 i8: %.0f us, %.0f TOP/s" % (us, 2 * 8192 ** 3 / us * 1e-6), flush=True)
    del x, y
    torch.cuda.empty_cache()
    for m, n, k, ld in ((8192, 8192, 8192, 8192), (4096, 4096, 4096, 4096), (4096, 4096, 4096, 4100), (4096, 4096, 4096, 4097), (777, 1003, 1289, 1289), (777, 1003, 1289, 1296),
                        (1024, 1024, 1008, 1008), (64, 4096, 4096, 4096), (128, 8192, 8192, 8192), (16, 4096, 4096, 4096), (1, 256, 1280, 1280), (512, 256, 1280, 1280)):
        product(torch.int8, m, n, k, ld)
    for dt in (torch.bfloat16, torch.float16):
        for m, n, k, ld in ((8192, 8192, 8192, 8192), (4096, 4096, 4096, 4096), (2048, 4096, 4096, 4096), (16, 4096, 4096, 4096), (41, 217, 3903, 3903), (41, 217, 3903, 3904)):
            product(dt, m, n, k, ld)
    product(torch.float32, 4096, 4096, 4096, 4096)
    for dt in (torch.int8, torch.float16):
        product(dt, 8192, 8192, 8192, 8192, zeros=True)


def product(dt, m, n, k, ld, zeros=False):
    """one product back to back, on operands that alternate where they are small"""
    import torch

    from pixelbox_amd import linear

    sets = []
    size = torch.empty((), dtype=dt).element_size()
    for _ in range(max(1, min(24, (1 << 28) // ((m + n) * ld * size)))):  # up to 256 MB of operands
        def rows(r):
            if dt == torch.int8:
                t = torch.randint(-127, 128, (r, ld), device="cuda", dtype=torch.int32).to(dt)
            else:
                t = torch.randn(r, ld, device="cuda").to(dt)
            return (t.zero_() if zeros else t)[:, :k]
        sets.append((rows(m), rows(n), torch.empty((m, n), dtype=torch.float16 if dt == torch.int8 else dt, device="cuda")))
    xs, ws, offsets, at = torch.ones(m, device="cuda"), torch.ones(n, device="cuda"), torch.tensor([0, m], dtype=torch.int32, device="cuda"), [0]

    def call():
        x, w, out = sets[at[0] % len(sets)]
        at[0] += 1
        if dt == torch.int8:
            linear.linear_i8(x, xs, w, ws, out=out)
        else:
            linear.linear_grouped(x, w.as_strided((1, n, k), (n * ld, ld, 1)), offsets, out=out)

    calls = 10 if m * n * k > 1 << 33 else 100
    g = torch.cuda.CUDAGraph()  # the device's time, not that of the checks of unusual strides
    for _ in range(2):
        call()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        for _ in range(calls):
            call()
    us = timed(g.replay, 1) / calls
    print("%s %d x %d x %d, rows of %d%s: %.1f us, %.0f T/s" % (dt, m, n, k, ld, ", zeros" if zeros else "", us, 2 * m * n * k / us * 1e-6), flush=True)


if __name__ == "__main__":
    what, rest = sys.argv[1], sys.argv[2:]
    if what == "trace":
        trace(rest[0])
    elif what == "counters":
        counters(rest)
    elif what == "time":
        time_all()
    elif what == "run":
        run(rest)
    else:
        import torch

        torch.cuda.set_stream(torch.cuda.Stream())
        h = Heads()
        for i8 in (False, True):
            for _ in range(15):
                h.with_heads(i8)
        torch.cuda.synchronize()
