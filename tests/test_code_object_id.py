"""The id of the stand-alone tracker code object is read from its file, without a device (TSDF_AQL=1 compares it)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "tracking_sdf_amd", "csrc")


def test_the_id_is_read_from_the_image_and_damaged_images_are_refused(tmp_path):
    exe = str(tmp_path / "elf_string_test")
    p = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-Wall", "-Wextra",
                        "-Werror", "-o", exe, os.path.join(ROOT, "tests", "host", "elf_string_test.cpp"), os.path.join(CSRC, "host_util.cpp"),
                        "-pthread", "-lrt"], capture_output=True, text=True, timeout=600)
    assert p.returncode == 0, p.stderr[-3000:]
    libdir = os.path.join(ROOT, "tracking_sdf_amd", "lib")
    p = subprocess.run([exe, os.path.join(libdir, "tsdf_track.hsaco"), "tsdf_track_build_id"], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-3000:]
    the_id = p.stdout.strip()
    assert len(the_id) == 32
    assert open(os.path.join(libdir, "libtsdf_hip.so"), "rb").read().count(the_id.encode()) >= 2     # host side and its own device code


def test_setting_the_queue_up_copies_nothing_to_existing_host_memory():
    """hsa_memory_copy to or from memory that HSA did not allocate page-locks it; the machines refuse that."""
    src = open(os.path.join(CSRC, "aql_queue.cpp")).read()
    assert "hsa_memory_copy" not in src and "hsa_amd_memory_lock" not in src
