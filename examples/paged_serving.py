"""Serving many requests over one paged cache: W1A8 linears and the paged operators.

A stack of attention layers at the benchmark model's width (hidden 2048, 16
query heads, 8 KV heads of 128) with seeded +-1 weights decodes requests of
unlike lengths together. Requests enter as others finish, pages go back to the
pool and out again, and one step may hold prompt chunks and single tokens. Per
layer:

  q|k|v linear   bnn_b200_execute_async, FP32 rows
  append         per-head norm, rotation, k and v to their pages
  attention      each request's new tokens over its pages, FP32 rows out
  o linear       bnn_b200_execute_async

Everything runs on the device handle's stream.

  python examples/paged_serving.py [--requests 24] [--layers 4] [--check]
"""
import argparse
import ctypes
import random
import sys
import time
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "bnn-train-infer_b200"))
from bnn_b200 import accel, paged, synth  # noqa: E402

HEADS, KV_HEADS, DIM, VOCAB, PAGE = 16, 8, 128, 512, 16
HIDDEN, KV = HEADS * DIM, KV_HEADS * DIM


class Rows:
    """An accelerator buffer and the float32 torch view of its device memory."""

    def __init__(self, dev, rows, width):
        self.buffer = accel.Buffer(dev, rows * width * 4)
        ptr = dev.api.dll.bnn_b200_buffer_device_ptr
        ptr.restype, ptr.argtypes = ctypes.c_void_p, [ctypes.c_void_p]
        self.__cuda_array_interface__ = {"data": (ptr(self.buffer.handle), False), "shape": (rows, width), "typestr": "<f4", "version": 3}
        self.t = torch.as_tensor(self, device="cuda")


class Stack:
    """The layers, and the linears as calls on the handle's stream."""

    def __init__(self, dev, layers, most_rows, seed=3):
        self.dev = dev
        rng = synth.rng_for(seed, salt=1)
        g = torch.Generator().manual_seed(seed)
        gain = lambda n: (1 + 0.1 * torch.randn(n, generator=g)).cuda()  # noqa: E731
        self.layers = [{"qkv": accel.Matrix(dev, *synth.w1_matrix(rng, HIDDEN, HIDDEN + 2 * KV)),
                        "o": accel.Matrix(dev, *synth.w1_matrix(rng, HIDDEN, HIDDEN)), "norm": gain(HIDDEN), "q_norm": gain(DIM),
                        "k_norm": gain(DIM)} for _ in range(layers)]
        self.embed = torch.randn(VOCAB, HIDDEN, generator=g).cuda()
        self.x, self.qkv = Rows(dev, most_rows, HIDDEN), Rows(dev, most_rows, HIDDEN + 2 * KV)
        self.y, self.o = Rows(dev, most_rows, HIDDEN), Rows(dev, most_rows, HIDDEN)
        freq = 1e6 ** (-torch.arange(DIM // 2, dtype=torch.float64) / (DIM // 2))
        angle = torch.arange(8192, dtype=torch.float64)[:, None] * freq
        self.cos, self.sin = angle.cos().float().cuda(), angle.sin().float().cuda()
        self._run = dev.api.dll.bnn_b200_execute_async
        self._run.restype, self._run.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(accel.Job)]

    def linear(self, matrix, src, dst, rows):
        job = accel.Job(operation=accel.OP_GEMM_F32, matrix=matrix.handle, input=accel.BufferView(src.buffer.handle, accel.TYPE_F32, 0, 0),
                        output=accel.BufferView(dst.buffer.handle, accel.TYPE_F32, 0, 0), rows=rows)
        st = self._run(self.dev.handle, ctypes.byref(job))
        if st != accel.OK:
            raise accel.BnnError(st, "bnn_b200_execute_async")

    def forward(self, ids, attend):
        """Hidden rows of the tokens; attend(layer index, layer, q, k, v, out) fills out with the attention."""
        t = len(ids)
        h = self.embed[ids]
        for i, layer in enumerate(self.layers):
            self.x.t[:t] = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * layer["norm"]
            self.linear(layer["qkv"], self.x, self.qkv, t)
            q, k, v = self.qkv.t[:t].view(t, -1, DIM).split((HEADS, KV_HEADS, KV_HEADS), 1)
            attend(i, layer, q, k, v, self.y.t[:t].view(t, HEADS, DIM))
            self.linear(layer["o"], self.y, self.o, t)
            h = h + self.o.t[:t]
        return h

    def free(self):
        torch.cuda.synchronize()
        for r in (self.x, self.qkv, self.y, self.o):
            r.buffer.free()
        for layer in self.layers:
            layer["qkv"].destroy()
            layer["o"].destroy()


class Server:
    """Pages, requests, steps."""

    def __init__(self, stack, ops, pages, most_batch, chunk):
        self.stack, self.ops, self.most_batch, self.chunk = stack, ops, most_batch, chunk
        shape = (len(stack.layers), pages, KV_HEADS, PAGE, DIM)
        self.k, self.v = (torch.empty(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.unused, self.running, self.waiting, self.done = list(range(pages)), [], [], []

    def submit(self, prompt, new_tokens):
        self.waiting.append({"ids": list(prompt), "prompt": len(prompt), "stop": len(prompt) + new_tokens, "kv": 0, "pages": []})

    def step(self):
        """One pass over everything that runs; returns the tokens that went through."""
        while self.waiting and len(self.running) < self.most_batch and \
                len(self.unused) * PAGE >= sum(r["stop"] + PAGE for r in self.running) + self.waiting[0]["stop"] + PAGE:
            self.running.append(self.waiting.pop(0))
        ids, positions, slots, starts, lens, tables = [], [], [], [0], [], []
        for r in self.running:
            n = min(self.chunk, len(r["ids"]) - r["kv"])
            while len(r["pages"]) * PAGE < r["kv"] + n:
                r["pages"].append(self.unused.pop())
            for p in range(r["kv"], r["kv"] + n):
                ids.append(r["ids"][p])
                positions.append(p)
                slots.append(r["pages"][p // PAGE] * PAGE + p % PAGE)
            r["kv"] += n
            starts.append(starts[-1] + n)
            lens.append(r["kv"])
            tables.append(r["pages"])
        width = max(map(len, tables))
        # one copy for the step's integers
        parts = [ids, positions, slots, starts, lens, [p for t in tables for p in t + [-1] * (width - len(t))]]
        flat = torch.from_numpy(np.concatenate([np.asarray(p, dtype=np.int32) for p in parts])).cuda(non_blocking=True)
        ids, positions, slots, starts_d, lens, table = flat.split([len(p) for p in parts])
        table = table.view(len(tables), width)
        max_q = max(b - a for a, b in zip(starts, starts[1:]))

        def attend(i, layer, q, k, v, out):
            q = self.ops.append(q, k, v, self.stack.cos, self.stack.sin, positions, slots, self.k[i], self.v[i], q_norm=layer["q_norm"],
                                k_norm=layer["k_norm"])
            self.ops.attention(q, self.k[i], self.v[i], table, lens, starts_d, max_q=max_q, out=out)

        h = self.stack.forward(ids, attend)
        last = h[starts_d[1:].long() - 1]
        logits = last @ self.stack.embed.T
        picks = logits.argmax(-1).tolist()
        still = []
        for r, pick, row in zip(self.running, picks, logits):
            if r["kv"] == len(r["ids"]):
                if len(r["ids"]) == r["stop"]:
                    r["logits"] = row
                    self.unused += r.pop("pages")
                    self.done.append(r)
                    continue
                r["ids"].append(pick)
            still.append(r)
        self.running = still
        return starts[-1]


def plain_logits(stack, ids):
    """The last logits of one request with plain attention over the whole of it."""
    def attend(i, layer, q, k, v, out):
        def turned(x, gain):
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gain
            a, b = x[..., :DIM // 2], x[..., DIM // 2:]
            c, s = stack.cos[:len(ids), None], stack.sin[:len(ids), None]
            return torch.cat((a * c - b * s, b * c + a * s), -1)
        q, k = turned(q, layer["q_norm"]).transpose(0, 1), turned(k, layer["k_norm"]).transpose(0, 1)
        k, v = (x.repeat_interleave(HEADS // KV_HEADS, 0) for x in (k, v.transpose(0, 1)))
        score = q @ k.transpose(1, 2) / DIM ** 0.5
        score.masked_fill_(torch.ones_like(score[0], dtype=torch.bool).triu(1), -torch.inf)
        out.copy_((score.softmax(-1) @ v).transpose(0, 1))

    return stack.forward(torch.tensor(ids, device="cuda"), attend)[-1] @ stack.embed.T


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=24)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--chunk", type=int, default=512, help="most prompt tokens of a request in one step")
    ap.add_argument("--longest", type=int, default=1500)
    ap.add_argument("--new", type=int, default=48)
    ap.add_argument("--check", action="store_true", help="compare each request's last logits with plain attention")
    a = ap.parse_args(argv)
    r = random.Random(5)
    dev = accel.Device(0)
    stream = dev.api.dll.bnn_b200_device_stream
    stream.restype, stream.argtypes = ctypes.c_void_p, [ctypes.c_void_p]
    with torch.cuda.stream(torch.cuda.ExternalStream(stream(dev.handle))), torch.no_grad():
        stack = Stack(dev, a.layers, max(a.batch * a.chunk, a.longest + a.new))
        ops = paged.Paged(dev, max_batch=a.batch)
        pages = a.batch * ((a.longest + a.new) // PAGE + 3) // 2 + (a.longest + a.new) // PAGE + 3
        server = Server(stack, ops, pages, a.batch, a.chunk)
        for _ in range(a.requests):
            n = r.randrange(1, a.longest + 1) if r.random() < 0.5 else r.randrange(1, 65)
            server.submit([r.randrange(VOCAB) for _ in range(n)], r.randrange(1, a.new + 1))
        torch.cuda.synchronize()
        began, steps, tokens = time.perf_counter(), 0, 0
        while server.running or server.waiting:
            tokens += server.step()
            steps += 1
        ops.sync()
        spent = time.perf_counter() - began
        made = sum(len(q["ids"]) - q["prompt"] for q in server.done)
        print(f"{len(server.done)} requests, {tokens} tokens through ({made} of them generated) in {steps} steps, {spent * 1e3:.1f} ms")
        worst = 0.0
        if a.check:
            for q in server.done:
                want = plain_logits(stack, q["ids"])
                worst = max(worst, float((q["logits"] - want).norm() / want.norm()))
            print(f"last logits against plain attention: relative difference at most {worst:.2g}")
        del server, ops
        stack.free()
    dev.close()
    return worst


if __name__ == "__main__":
    main()
