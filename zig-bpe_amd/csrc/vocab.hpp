// Host side of the grammar operators: the bytes of a vocabulary's tokens.
#pragma once
#include <stdint.h>

#include <string>
#include <vector>

#include "../../include/zbpe.h"

namespace zbpe {

// The tokens' lengths and an order in which every token comes after its halves (decode's rules: a token below 256 is its
// byte, any other the first merge that makes it). Iterative: a table read from a file may nest as deep as it is long.
struct VocabTree {
    struct Node {
        int32_t a = -1, b = -1;  // halves; -1: no merge makes this id
    };
    std::vector<Node> node;
    std::vector<uint64_t> len;
    std::vector<uint32_t> order;  // ids from 256 on that have bytes, halves first
    uint64_t total = 0;
    std::string err;

    zbpe_status build(const uint16_t *triples, size_t n_merges, size_t vocab_size) {
        node.assign(vocab_size, Node{});
        len.assign(vocab_size, 0);
        for (size_t v = 0; v < 256; v++) len[v] = 1;
        for (size_t i = 0; i < n_merges; i++) {
            const uint16_t *t = triples + 3 * i;
            if (t[2] >= vocab_size) {
                err = "merge " + std::to_string(i) + " makes token " + std::to_string(t[2]) + ", outside a vocabulary of " + std::to_string(vocab_size);
                return ZBPE_INVALID_ARGUMENT;
            }
            if (t[2] < 256 || node[t[2]].a >= 0) continue;
            node[t[2]] = Node{t[0], t[1]};
        }
        constexpr uint64_t MOST = (1ull << 31) - 1;
        std::vector<uint8_t> open(vocab_size, 0);  // 1: on the path from the root, 2: done
        std::vector<uint32_t> path;
        for (size_t v = 256; v < vocab_size; v++) {
            if (node[v].a < 0 || open[v] == 2) continue;
            path.push_back((uint32_t)v);
            while (!path.empty()) {
                const uint32_t x = path.back();
                open[x] = 1;
                uint32_t child = 0;
                for (int32_t h : {node[x].a, node[x].b}) {
                    if (h < 256) continue;
                    const bool made = (size_t)h < vocab_size && node[h].a >= 0;
                    if (!made || open[h] == 1) {
                        err = "token " + std::to_string(x) + " is made from token " + std::to_string(h) +
                              (made ? ", which is made from it" : ", which no merge makes");
                        return ZBPE_INVALID_TOKEN;
                    }
                    if (open[h] == 2) continue;
                    child = (uint32_t)h;
                    break;
                }
                if (child) {
                    path.push_back(child);
                    continue;
                }
                len[x] = len[node[x].a] + len[node[x].b];
                if (len[x] > MOST) {
                    err = "token " + std::to_string(x) + " has 2^31 bytes or more";
                    return ZBPE_INVALID_ARGUMENT;
                }
                open[x] = 2;
                order.push_back(x);
                path.pop_back();
            }
        }
        for (uint64_t l : len) total += l;
        if (total > MOST) {
            err = "the tokens have 2^31 bytes or more";
            return ZBPE_INVALID_ARGUMENT;
        }
        return ZBPE_OK;
    }

    void write(uint32_t *offsets, uint8_t *bytes) const {
        uint64_t at = 0;
        for (size_t v = 0; v < len.size(); v++) {
            offsets[v] = (uint32_t)at;
            at += len[v];
        }
        offsets[len.size()] = (uint32_t)at;
        if (!bytes) return;
        for (size_t v = 0; v < 256; v++) bytes[offsets[v]] = (uint8_t)v;
        for (uint32_t v : order) {
            uint8_t *to = bytes + offsets[v];
            const uint32_t a = (uint32_t)node[v].a, b = (uint32_t)node[v].b;
            for (uint64_t i = 0; i < len[a]; i++) to[i] = bytes[offsets[a] + i];
            for (uint64_t i = 0; i < len[b]; i++) to[len[a] + i] = bytes[offsets[b] + i];
        }
    }
};

}  // namespace zbpe
