"""The optimizer's host side without a GPU: the C call of a step is taken over by the formula in numpy, which reads the table and the
addresses that the kernel would."""
import ctypes
import struct

import numpy as np
import torch as ch

BLOCK = 256


def at(address, n, kind):
    """n values of memory."""
    size = np.dtype(kind).itemsize
    return np.frombuffer((ctypes.c_char * (n * size)).from_address(address), kind) if n else np.zeros(0, kind)


class HostLibrary:
    """Stands for ``libffcv_b200.so``: the host's functions are its own, a step is made here.  ``steps`` counts them, ``grads`` has the last
    one's addresses of gradients."""

    def __init__(self, lib, native):
        self.lib, self.native, self.steps, self.grads = lib, native, 0, None

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def ffcvb_adamw_step(self, args, numel, steps, group_of, grads, groups, n_groups, stream):
        self.steps += 1
        table, m_at, v_at, scales_at, master_at, norm_at, _, seed, _, kind, bits, n, max_norm = self.native.ADAMW.unpack(args)
        assert max_norm == 0.0
        self.grads = list(struct.unpack(f'={n}Q', grads))
        grads, numel, steps, group_of = struct.unpack(f'={n}Q', grads), at(numel, n, np.int64), at(steps, n, np.int64), at(group_of, n, np.int32)
        tensors = at(table, 3 * n, np.int64).reshape(n, 3)
        for i, (param, count, start) in enumerate(tensors.tolist()):
            assert count == numel[i]
            if not grads[i]:
                continue
            steps[i] += 1
            lr, b1, b2, eps, decay = self.native.ADAMW_GROUP.unpack_from(groups, int(group_of[i]) * 40)
            t = int(steps[i])
            w, g = self.values(param, count, kind), self.values(grads[i], count, kind).astype(np.float64)
            master = w if kind == 0 else at(master_at + 4 * start, count, np.float32)
            m, v = self.moment(m_at, scales_at, 0, start, count, bits), self.moment(v_at, scales_at, 1, start, count, bits)
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
            master[:] = master * (1 - lr * decay) - lr * m / (1 - b1 ** t) / (np.sqrt(v / (1 - b2 ** t)) + eps)
            if kind:
                self.values(param, count, kind, master)
            for where, k, new in ((m_at, 0, m), (v_at, 1, v)):
                self.moment(where, scales_at, k, start, count, bits, new)
        return 0

    def ffcvb_adamw_masters(self, args, numel, which, stream):
        table, _, _, _, master_at, _, _, _, _, kind, _, n, _ = self.native.ADAMW.unpack(args)
        which, tensors = struct.unpack(f'={n}Q', which), at(table, 3 * n, np.int64).reshape(n, 3)
        dtype = (None, ch.float16, ch.bfloat16)[kind]
        for (param, count, start), asked in zip(tensors.tolist(), which):
            if asked:
                w, master = self.values(param, count, kind), at(master_at + 4 * start, count, np.float32)
                rounded = ch.from_numpy(master.copy()).to(dtype).float().numpy()
                master[:] = np.where(rounded == w, master, w)
        return 0

    @staticmethod
    def values(address, n, kind, new=None):
        if kind == 0:
            return at(address, n, np.float32)
        dtype = (None, ch.float16, ch.bfloat16)[kind]
        raw = at(address, n, np.uint16)
        if new is not None:
            raw[:] = ch.from_numpy(np.ascontiguousarray(new)).to(dtype).view(ch.uint16).numpy()
        return ch.from_numpy(raw.copy()).view(dtype).float().numpy()

    @staticmethod
    def moment(address, scales_at, k, start, n, bits, new=None):
        """A tensor's part of a flat moment; with `new`, that is written (8 bits: rounded to the nearest)."""
        if bits == 32:
            flat = at(address + 4 * start, n, np.float32)
            if new is not None:
                flat[:] = new
            return flat.astype(np.float64)
        dtype, top = ((ch.float8_e4m3fn, 7), (ch.float8_e5m2, 14))[k]
        blocks = -(-n // BLOCK)
        raw, scales = at(address + start, n, np.uint8), at(scales_at + start // BLOCK * 8, 2 * blocks, np.float32)[k::2]
        if new is not None:
            padded = np.zeros((blocks, BLOCK))
            padded.reshape(-1)[:n] = new
            power = np.maximum(np.frexp(np.abs(padded).max(1))[1] - 1, -126)
            scales[:] = np.ldexp(1.0, power - top)
            scaled = np.ldexp(padded, (top - power)[:, None]).reshape(-1)[:n].astype(np.float32)
            raw[:] = ch.from_numpy(scaled).to(dtype).view(ch.uint8).numpy()
        return ch.from_numpy(raw.copy()).view(dtype).float().numpy().astype(np.float64) * np.repeat(scales, BLOCK)[:n]


def on_the_host(monkeypatch):
    """An AdamW for tensors of the CPU, and its library."""
    from ffcv_b200.training import AdamW
    from ffcv_b200.training import _native as N
    lib = HostLibrary(N.lib, N)
    monkeypatch.setattr(N, 'lib', lib)
    monkeypatch.setattr(N, 'raw_stream', lambda index: 0)
    monkeypatch.setattr(N, 'capturing', lambda: False, raising=False)
    monkeypatch.setattr(N, 'require', lambda tensor, name, like=None: N.TYPES[tensor.dtype])
    return AdamW, lib
