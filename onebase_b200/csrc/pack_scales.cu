// One-time re-layout of an NVFP4 weight's ue4m3 block scales: linear [N, K/16] (the checkpoint's layout) -> the order in
// which K2 moves them to TMEM; and of an MXFP4 weight's scale bytes [N, K/32], with two atoms per K slot instead of four.  Per (128-row output tile of a slice, 256-element K slot) 2048 bytes = 4 atoms (one per
// 64-element MMA) of 512 bytes [row % 32][row / 32][4 scales]: the scale-factor atom of the block-scaled tcgen05 MMA.
// Rows past a slice's width and scale columns past K/16 are zero.
#include "ob_common.cuh"

namespace ob {

struct PackArgs {
    int cols, kslots, S;   // scales of a row: K/16 or K/32
    int atoms_log;         // atoms per K slot: 4 (NVFP4) or 2 (MXFP4)
    int widths[OB_MAX_SLICES];
};

__global__ void pack_scales_kernel(const uint8_t* __restrict__ linear, uint8_t* __restrict__ packed, size_t bytes, PackArgs a) {
    for (size_t o = blockIdx.x * (size_t)blockDim.x + threadIdx.x; o < bytes; o += (size_t)gridDim.x * blockDim.x) {
        const int j = (int)(o & 3), r4 = (int)((o >> 2) & 3), r32 = (int)((o >> 4) & 31), m = (int)(o >> 9) & ((1 << a.atoms_log) - 1);
        const size_t slot = o >> (9 + a.atoms_log);
        const int kb = (int)(slot % a.kslots);
        int tile = (int)(slot / a.kslots), s = 0, row0 = 0;
        while (s < a.S - 1 && tile >= (a.widths[s] + kTileN - 1) / kTileN) {
            tile -= (a.widths[s] + kTileN - 1) / kTileN;
            row0 += a.widths[s];
            ++s;
        }
        const int r = tile * kTileN + r4 * 32 + r32, col = (kb << (2 + a.atoms_log)) + m * 4 + j;
        packed[o] = (r < a.widths[s] && col < a.cols) ? linear[(size_t)(row0 + r) * a.cols + col] : (uint8_t)0;
    }
}

// A launch without work, and without the programmatic attribute: it starts when everything before it in the stream is complete and visible,
// and a projection behind it -- whose kernels read weights, scales and adapters before their wait on the preceding launch -- starts behind
// it.  (Directly behind the kernel that wrote an operand, a programmatic dependent may start when that kernel's CTAs have left, and only its
// wait makes what they wrote visible.)
__global__ void operand_fence_kernel() {}

cudaError_t launch_operand_fence(cudaStream_t stream) {
    operand_fence_kernel<<<1, 1, 0, stream>>>();
    return cudaGetLastError();
}

cudaError_t launch_pack_scales(int base_fmt, const uint8_t* linear, int K, int S, const int32_t* widths, uint8_t* packed, size_t bytes,
                               cudaStream_t stream) {
    PackArgs a = {};
    a.atoms_log = base_fmt == OB_BASE_MXFP4 ? 1 : 2;
    a.cols = K / (64 >> a.atoms_log);
    a.kslots = (K + 255) / 256;
    a.S = S;
    for (int s = 0; s < S; ++s) a.widths[s] = widths[s];
    const int threads = 256;
    size_t blocks = (bytes + threads - 1) / threads;
    if (blocks > 148 * 32) blocks = 148 * 32;
    pack_scales_kernel<<<(unsigned)blocks, threads, 0, stream>>>(linear, packed, bytes, a);
    return cudaGetLastError();
}

}  // namespace ob
