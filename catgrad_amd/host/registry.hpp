// The models this driver knows, by what a model folder's config.json says: "architecture" (or the "model_type" /
// "architectures" of a Llama or Qwen3 checkpoint).
#pragma once

#include <memory>

#include "loretar.hpp"
#include "lufatar.hpp"
#include "models.hpp"

namespace cgh {

// How a checkpoint says that its positions' frequencies are scaled (rope.rs:8-62); "default" and none: not at all.
inline void read_rope_scaling(const Json &j, cg_rotation &r) {
    const Json *s = j.find("rope_scaling"), *t = s ? s->find("rope_type") : nullptr;
    if (s && !t) t = s->find("type");
    if (!s || !t || t->str() == "default") return;
    auto value = [&](const char *name, double otherwise) {
        const Json *v = s->find(name);
        return v ? v->real() : otherwise;
    };
    r.factor = s->at("factor").real();
    if (t->str() == "linear") r.scaling = CG_ROTATION_LINEAR;
    else if (t->str() == "llama3" || t->str() == "yarn") {
        const bool bands = t->str() == "llama3";
        const Json *all = j.find("max_position_embeddings");
        r.scaling = bands ? CG_ROTATION_BANDS : CG_ROTATION_RAMP;
        r.low = bands ? s->at("low_freq_factor").real() : value("beta_slow", 1.0);
        r.high = bands ? s->at("high_freq_factor").real() : value("beta_fast", 32.0);
        r.original = value("original_max_position_embeddings", all ? all->real() : 0.0);
        if (!bands) { // (what else the section may say about its limits and its magnitude is refused, not passed over)
            const Json *whole = s->find("truncate");
            r.magnitude = value("attention_factor", 0.0);
            if (whole && !whole->flag()) throw ConfigError("config: rope_scaling's limits are whole pairs (\"truncate\")");
            if (r.magnitude == 0.0 && (value("mscale", 0.0) != 0.0 || value("mscale_all_dim", 0.0) != 0.0))
                throw ConfigError("config: rope_scaling's \"mscale\" is not followed; \"attention_factor\" is");
        }
    } else {
        throw ConfigError("config: unknown rope_scaling '" + t->str() + "'");
    }
}
// "kv_cache": "f8" has keys and values held as 8-bit codes, with scaled frequencies where "rope_scaling" asks for them; "f32": as ever.
inline void read_cache(const Json &j, const std::string &kind, LlmConfig &c) {
    if (kind == "f32") return;
    if (kind != "f8") throw ConfigError("config: kv_cache is \"f32\" or \"f8\"");
    if (c.head_dim < 16 || c.head_dim > 256 || c.head_dim % 16) throw ConfigError("config: an 8-bit cache holds heads of 16, 32, .. 256 channels");
    c.cache8 = true;
    c.rotation.dims = c.head_dim;
    c.rotation.base = c.rope_theta;
    read_rope_scaling(j, c.rotation);
}

// llama.rs:13-60, qwen3.rs:14-60: the fields the dense graphs read
inline LlmConfig read_llm_config(const Json &j, int arch) {
    LlmConfig c;
    c.arch = arch;
    c.hidden_size = j.at("hidden_size").nat();
    c.num_hidden_layers = j.at("num_hidden_layers").nat();
    c.num_attention_heads = j.at("num_attention_heads").nat();
    const Json *kv = j.find("num_key_value_heads"), *hd = j.find("head_dim"), *tie = j.find("tie_word_embeddings");
    c.num_key_value_heads = kv ? kv->nat() : c.num_attention_heads;
    if (!c.num_attention_heads || !c.num_key_value_heads) throw ConfigError("config: no attention heads");
    c.head_dim = hd ? hd->nat() : c.hidden_size / c.num_attention_heads;
    c.intermediate_size = j.at("intermediate_size").nat();
    c.vocab_size = j.at("vocab_size").nat();
    c.rms_norm_eps = (float)j.at("rms_norm_eps").real();
    c.rope_theta = (float)j.at("rope_theta").real();
    c.tie_word_embeddings = tie && tie->flag();
    if (const Json *k = j.find("kv_cache")) read_cache(j, k->str(), c);
    return c;
}

// weights: CG_F32, or CG_BF16 for matrices at bfloat16 precision (models that have such a form)
inline std::unique_ptr<Model> make_model(Interpreter &i, const Json &config, cg_dtype weights) {
    std::string name;
    if (const Json *a = config.find("architecture")) name = a->str();
    else if (const Json *t = config.find("model_type")) name = t->str();
    else if (const Json *l = config.find("architectures"))
        if (!l->list().empty()) name = l->list()[0].str();
    const Json *cache = config.find("kv_cache");
    if ((name == "Loretar" || name == "Lufatar") && cache && cache->str() != "f32") throw ConfigError("config: kv_cache \"f8\" is for Llama and Qwen3");
    if (name == "Loretar") return std::make_unique<LoretarModel>(i, LoretarConfig::read(config), weights);
    if (name == "Lufatar") return std::make_unique<LufatarModel>(i, LufatarConfig::read(config), weights);
    int arch = name == "llama" || name == "LlamaForCausalLM" ? 0 : name == "qwen3" || name == "Qwen3ForCausalLM" ? 1 : -1;
    if (arch < 0) throw ConfigError("config: unknown architecture '" + name + "'");
    if (weights != CG_F32) throw ConfigError("config: this architecture runs in f32 only");
    LlmConfig c = read_llm_config(config, arch);
    if (c.cache8) i.backend.check_rotation(c.rotation);
    return std::make_unique<LlmModel>(i, c);
}

} // namespace cgh
