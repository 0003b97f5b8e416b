"""The output area of a frame sharded over processes: a shared-memory segment that is ordinary memory to every process's
GPU.  Each process's sections pass through its context's own page-locked buffer, so the form has to work where
page-locking memory that already exists is refused.  Expected bytes: the oracle's whole-frame codestream."""
import multiprocessing as mp
import os
import subprocess

import numpy as np
import pytest

import jxlt_testlib as T


def test_the_host_library_page_locks_nothing_that_it_does_not_own(built):
    lib = T.ROOT / "libjxl-tiny_amd" / "host" / "libjxltiny_host.so"
    wanted = subprocess.run(["nm", "-D", "--undefined-only", str(lib)], capture_output=True, text=True, check=True).stdout
    assert "jxlt_pinned_alloc" in wanted and "jxlt_output_buffer" in wanted
    assert "jxlt_pinned_register" not in wanted and "HostRegister" not in wanted


def test_a_segment_that_the_file_system_has_no_room_for_is_refused(built):
    """... when it is opened, not by a signal when somebody's sections reach a page that is not there."""
    fs = os.statvfs("/dev/shm")
    if fs.f_blocks == 0:
        pytest.skip("/dev/shm has no limit here")
    name = "/jxlt-no-room-%d" % os.getpid()
    with pytest.raises(built.JxlTinyError):
        built.ShardGroup(name, 0, 2, fs.f_blocks * fs.f_frsize + (1 << 30), 4096)
    assert not os.path.exists("/dev/shm" + name)
    grp = built.ShardGroup(name, 0, 1, 1 << 20, 4096)
    segment = os.stat("/dev/shm" + name)
    assert segment.st_size > 1 << 20 and segment.st_blocks * 512 >= segment.st_size  # (every page is there)
    grp.close()


def _slab(planes, rect):
    x0, y0, x1, y1 = rect
    return np.ascontiguousarray(planes[:, y0:y1, x0:x1])


def _group_rank(pkg, name, rank, world, frames, barrier):
    """The frames in turn through one group; the rank's codestreams (None on the ranks that hold none)."""
    enc = pkg.Encoder(0)
    grp = pkg.ShardGroup(name, 0, world, 8 << 20, 4096) if rank == 0 else None
    barrier.wait()
    if grp is None:
        grp = pkg.ShardGroup(name, rank, world, 8 << 20, 4096)
    out = []
    for w, h, d in frames:
        rect = pkg.shard_rect(w, h, world, rank)
        if rect[3] > rect[1]:
            enc.upload(_slab(T.to_planes(T.synthetic_image(w, h)), rect))
        v = grp.encode(enc, w, h, d)
        out.append(v.tobytes() if v is not None else None)
    barrier.wait()
    grp.close()
    enc.close()
    return out


def _pipeline_rank(pkg, name, rank, world, frames, barrier):
    """The frames, resident in device memory, with two of them in flight."""
    import torch
    pipe = pkg.ShardPipeline(name, 0, world, 0, 2, 8 << 20, 4096) if rank == 0 else None
    barrier.wait()
    if pipe is None:
        pipe = pkg.ShardPipeline(name, rank, world, 0, 2, 8 << 20, 4096)
    slabs, tickets, out = [], [], []
    take = lambda v: out.append(v.tobytes() if v is not None else None)
    for k, (w, h, d) in enumerate(frames):
        rect = pkg.shard_rect(w, h, world, rank)
        t = torch.from_numpy(_slab(T.to_planes(T.synthetic_image(w, h)), rect)).cuda()
        torch.cuda.synchronize()
        slabs.append(t)
        if k >= 2:
            take(pipe.wait(tickets[k - 2]))
        empty = t.numel() == 0
        tickets.append(pipe.submit_device(None if empty else [t[c].data_ptr() for c in range(3)], t.shape[2] * 4, w, h,
                                          0 if empty else t.shape[1], d))
    for tk in tickets[-2:]:
        take(pipe.wait(tk))
    barrier.wait()
    pipe.close()
    return out


def _process(form, name, rank, world, frames, barrier, q):
    try:
        q.put((rank, {"group": _group_rank, "pipeline": _pipeline_rank}[form](T.product(), name, rank, world, frames, barrier)))
    except Exception as e:  # pragma: no cover
        barrier.abort()
        q.put((rank, "ERROR: %r" % (e,)))


def _run(form, world, frames):
    ctx = mp.get_context("spawn")
    q, barrier = ctx.Queue(), ctx.Barrier(world)
    name = "/jxlt-%s-%d" % (form, os.getpid())
    procs = [ctx.Process(target=_process, args=(form, name, r, world, frames, barrier, q)) for r in range(world)]
    for p in procs:
        p.start()
    results = dict(q.get(timeout=100) for _ in range(world))
    for p in procs:
        p.join(timeout=30)
    return results


# a frame cut along its columns (three DC groups in a row: the AC sections of a slab are three runs of the codestream),
# one cut along its rows (one run), the first again (the staging buffer has grown in between), a participant without work
FRAMES = [(2 * 2048 + 4, 600, 1.0), (600, 2 * 2048 + 520, 0.5), (2 * 2048 + 4, 600, 1.0), (2048 + 40, 264, 2.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("form,world", [("group", 2), ("group", 3), ("pipeline", 2)])
def test_processes_on_one_gpu_give_the_whole_frame(built, form, world):
    results = _run(form, world, FRAMES)
    want = {}
    for w, h, d in set(FRAMES):
        want[w, h, d] = T.assemble_codestream(T.oracle_hot_path(T.to_planes(T.synthetic_image(w, h)), d), d)
    assert isinstance(results[0], list), results[0]
    for k, f in enumerate(FRAMES):
        assert results[0][k] == want[f], (k, f)
    for r in range(1, world):
        assert results[r] == [None] * len(FRAMES), (r, results[r] if isinstance(results[r], str) else "bytes")
